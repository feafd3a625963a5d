"""Measured cases of the operators that serve a compressed model: the matrix product with 4-bit weights, the write into an
8-bit paged cache, and the attention over that cache.  Every case runs either in plain torch (`own` false) or through
the package's entry points (`own` true) on the same inputs."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CACHE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
HALF_RANGE = {"e4m3": 448.0, "int8": 127.5}  # half of the code range: the symmetric min-max scale is absmax over this
EPS = 2.0 ** -23  # smallest scale the package's calibration gives
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------------------------- cases

def _linear(name, tokens, rows, cols, codec="int4", group=128, zp=False, bias=False, dtype="bf16"):
    return dict(name=name, op="linear", tokens=tokens, rows=rows, cols=cols, codec=codec, group=group, zp=zp, bias=bias, dtype=dtype)


def _append(name, batch, new, history, heads=8, dim=128, block=64, cache="e4m3", dtype="bf16", lens=1):
    return dict(name=name, op="append", batch=batch, new=new, history=history, heads=heads, dim=dim, block=block, cache=cache,
                dtype=dtype, lens=lens)


def _attend(name, batch, context, queries=1, q_heads=32, heads=8, dim=128, block=64, cache="e4m3", dtype="bf16", lens=1):
    return dict(name=name, op="attend", batch=batch, context=context, queries=queries, q_heads=q_heads, heads=heads, dim=dim,
                block=block, cache=cache, dtype=dtype, lens=lens)


def listed():
    return [
        # one token through the k / v projection of a Llama-3-8B layer: the smallest product, where latency counts
        _linear("int4 kv_proj 1 token", 1, 1024, 4096),
        # one token through the widest projection of that layer
        _linear("int4 down_proj 1 token", 1, 4096, 14336),
        # a small batch of decoding requests through the gate projection
        _linear("int4 gate_proj 16 tokens", 16, 14336, 4096),
        # asymmetric codes in small groups, float16, sizes that are no multiple of a tile
        _linear("int4 zp g32 odd f16", 5, 2999, 2080, group=32, zp=True, bias=True, dtype="f16"),
        # NVFP4 weights (e4m3 scales per 16 columns, a global scale), eight decoding requests
        _linear("nvfp4 gate_proj 8 tokens", 8, 14336, 4096, codec="nvfp4", group=16),
        # one new token per request of a decoding batch, into blocks that already hold tokens
        _append("append decode 64", 64, 1, 100, cache="int8", lens=2),
        # four prompts written whole
        _append("append prompts", 4, 4096, 0, lens=3),
        # a single short request: the smallest attention
        _attend("attend 1 x 200", 1, 200, lens=4),
        # a single request with a long context: the cache has to be split to fill the GPU
        _attend("attend 1 x 32768", 1, 32768, lens=5),
        # a decoding batch with ragged contexts, float16, small blocks, int8 codes, head size 64
        _attend("attend 16 ragged int8", 16, 3001, q_heads=16, heads=4, dim=64, block=16, cache="int8", dtype="f16", lens=6),
        # a full decoding batch: the largest cache
        _attend("attend 64 ragged", 64, 8192, lens=7),
        # chunks of two prompts against what is cached of them
        _attend("attend prompt chunks", 2, 4096, queries=512, lens=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "append", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    lens = rng.randrange(1 << 20)
    if op == "linear":
        codec = rng.choice(("int4", "int4", "nvfp4"))
        group = 16 if codec == "nvfp4" else rng.choice((32, 64, 128, 128, -1))
        step = max(group, 32)
        case = _linear("", _log(rng, 1, 32), _log(rng, 64, 14336), step * _log(rng, max(1, 256 // step), 14336 // step), codec, group,
                       codec == "int4" and rng.random() < 0.4, rng.random() < 0.3, dtype)
    elif op == "append":
        prompts = rng.random() < 0.5
        new = _log(rng, 2, 4096) if prompts else 1
        case = _append("", _log(rng, 1, min(256, 16384 // new)), new, rng.choice((0, _log(rng, 1, 300))), rng.choice((1, 2, 4, 8)),
                       rng.choice((64, 128, 128, 256)), rng.choice((16, 32, 64, 128)), rng.choice(("e4m3", "int8")), dtype, lens)
    else:
        heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, 256))
        q_heads = heads * rng.choice((1, 2, 4, 4, 7, 8))
        kind = rng.random()
        queries = 1 if kind < 0.6 else _log(rng, 2, 8) if kind < 0.8 else _log(rng, 9, 512)
        context = max(queries, _log(rng, 1, 32768 if queries == 1 else 4096))
        most = 2 ** 29 // (context * heads * dim)  # elements of the keys
        if queries > 1:
            most = min(most, 2 ** 27 // (q_heads * queries * context))
        case = _attend("", _log(rng, 1, max(1, min(64, most))), context, queries, q_heads, heads, dim, rng.choice((16, 32, 64, 128)),
                       rng.choice(("e4m3", "int8")), dtype, lens)
    del case["name"]
    return case


def _lens(case):
    """(tokens in the cache after the call, tokens of the call) per request: ragged, part of the case."""
    rng = random.Random(case["lens"])
    out = []
    for i in range(case["batch"]):
        if case["op"] == "append":
            new = case["new"] if case["new"] == 1 or i == 0 else rng.randint(max(1, case["new"] // 2), case["new"])
            out.append((new + (rng.randint(case["history"] // 2, case["history"]) if case["history"] else 0), new))
        else:
            new = case["queries"] if i == 0 else rng.randint((case["queries"] + 1) // 2, case["queries"])
            total = case["context"] if i == 0 else rng.randint(case["context"] // 8, case["context"])
            out.append((total if case["queries"] == 1 else max(total, new), new))
    return out


# --------------------------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _generator(seed)
    return _prepare_linear(case, g) if case["op"] == "linear" else _prepare_cache(case, g)


def _prepare_linear(case, g):
    n, k, dt = case["rows"], case["cols"], DTYPES[case["dtype"]]
    group = k if case["group"] == -1 else case["group"]
    s = dict(case=case, group=group, zp=None, gs=None, bias=None)
    s["x"] = torch.randn(case["tokens"], k, generator=g, device="cuda").to(dt)
    if case["codec"] == "int4":  # bell-shaped codes, as a calibrated weight has them
        codes = torch.empty(n, k, dtype=torch.float16, device="cuda").normal_(0.0, 2.7, generator=g).round_().clamp_(-8, 7).to(torch.int32)
        words = torch.zeros(n, -(-k // 8), dtype=torch.int32, device="cuda")
        for i in range(8):
            part = codes[:, i::8] + 8
            words[:, :part.shape[1]] |= part << (4 * i)
        s["q"] = words
        s["scale"] = (torch.rand(n, k // group, generator=g, device="cuda") * 0.01 + 0.002).to(dt)
        if case["zp"]:
            s["zp"] = torch.randint(-8, 8, (n, k // group), generator=g, device="cuda", dtype=torch.int8)
    else:
        s["q"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scale"] = (torch.rand(n, k // group, generator=g, device="cuda") * 400 + 8).to(torch.float8_e4m3fn)
        s["gs"] = torch.full((1,), 448.0 * 6 / 0.15, device="cuda")
    if case["bias"]:
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(dt)
    return s


def _prepare_cache(case, g):
    lens = _lens(case)
    total, new = [a for a, _ in lens], [b for _, b in lens]
    block, heads, dim, dt, cdt = case["block"], case["heads"], case["dim"], DTYPES[case["dtype"]], CACHE[case["cache"]]
    width = max(1, -(-max(total) // block))
    used = [-(-t // block) for t in total]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).tolist()
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):  # every request owns its pages; what lies behind them in the table is never read
        table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
        at += u
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    tokens = starts[-1]
    s = dict(case=case, table=table.cuda(), seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"),
             query_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_len=max(total), max_new=max(new))
    owner = torch.tensor([b for b, m in enumerate(new) for _ in range(m)], device="cuda")
    place = torch.tensor([j for m in new for j in range(m)], device="cuda")
    s["owner"], s["place"] = owner, place
    for name in ("k", "v"):
        cache = torch.empty(pages, heads, block, dim, dtype=cdt, device="cuda")
        scale = (torch.rand(pages, heads, generator=g, device="cuda") + 0.5) * (4.0 / HALF_RANGE[case["cache"]])
        for i in range(0, pages, 512):  # values of unit variance under scales that differ from block to block
            x = torch.randn(cache[i:i + 512].shape, generator=g, device="cuda") / scale[i:i + 512, :, None, None]
            x = x.clamp_(-448, 448) if cdt is not torch.int8 else x.round_().clamp_(-128, 127)
            cache[i:i + 512] = x.to(cdt)
        s[name + "_cache"], s[name + "_scale"] = cache, scale
    # queries, keys and values as one fused projection leaves them
    q_heads = case.get("q_heads", heads)
    fused = torch.randn(tokens, q_heads + 2 * heads, dim, generator=g, device="cuda").to(dt)
    s["q"], s["k"], s["v"] = fused[:, :q_heads], fused[:, q_heads:q_heads + heads], fused[:, q_heads + heads:]
    return s


# ------------------------------------------------------------------------------------------------------------------ run

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[op](state)


def _own(op, s):
    from compressed_tensors_b200 import torch_ops as ops

    if op == "linear":
        nvfp4 = s["case"]["codec"] == "nvfp4"
        return ops.dequantize_linear(s["x"], s["q"], s["scale"], s["zp"], qtype=ops.QFLOAT if nvfp4 else ops.QINT, bits=4,
                                     col_group=s["group"], scale_row_stride=s["scale"].shape[1], codec="fp4x2" if nvfp4 else "pack32",
                                     global_scale=s["gs"], bias=s["bias"])
    if op == "append":
        ops.kv_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"],
                            s["query_start"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    return list(ops.kv_cache_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"],
                                       s["query_start"], return_lse=True))


def _plain_linear(s):
    case, x, q, scale = s["case"], s["x"], s["q"], s["scale"].float()
    n, k = case["rows"], case["cols"]
    if case["codec"] == "int4":
        shifts = torch.arange(0, 32, 4, device=q.device, dtype=torch.int32)
        codes = ((q[:, :, None] >> shifts) & 15).reshape(n, -1)[:, :k].float() - 8.0
    else:
        both = torch.stack((q & 15, q >> 4), dim=-1).reshape(n, k).long()
        codes = torch.tensor(E2M1, device=q.device)[both & 7]
        codes = torch.where(both > 7, -codes, codes)
        scale = scale / s["gs"]
    codes = codes.reshape(n, scale.shape[1], -1)
    if s["zp"] is not None:
        codes = codes - s["zp"].float()[:, :, None]
    w = (codes * scale[:, :, None]).reshape(n, k)
    y = x.float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def _to_codes(x, kind):
    """Exact quotients (64 bits) onto the nearest value of the code grid, ties to the even code."""
    if kind == "int8":
        return x.round().clamp(-128, 127).to(torch.int8)
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)  # three bits behind the leading one; 2^-9 below 2^-6
    return ((x / step).round() * step).clamp(-448, 448).float().to(torch.float8_e4m3fn)


def _plain_append(s):
    case = s["case"]
    block, kind = case["block"], case["cache"]
    owner, place = s["owner"], s["place"]
    new = (s["query_start"][1:] - s["query_start"][:-1]).long()
    first = (s["seq_lens"].long() - new)  # position of each request's first new token
    position = first[owner] + place
    page = s["table"].long()[owner, position // block]
    slot = position % block
    # the block that a request's first new token falls into may hold earlier tokens of the request: those are kept
    kept = torch.zeros(s["k_cache"].shape[0], dtype=torch.long, device=page.device)
    kept[s["table"].long()[torch.arange(len(first), device=page.device), first // block]] = first % block
    touched = torch.zeros_like(kept, dtype=torch.bool)
    touched[page] = True
    for name in ("k", "v"):
        x, cache, scale = s[name].double(), s[name + "_cache"], s[name + "_scale"]
        most = torch.zeros_like(scale, dtype=torch.float64)
        most.index_reduce_(0, page, x.abs().amax(dim=2), "amax")
        now = (most / HALF_RANGE[kind]).float().clamp(min=EPS)
        now = torch.where((kept > 0)[:, None], torch.maximum(scale, now), now)
        grown = touched[:, None] & (kept > 0)[:, None] & (now > scale)
        old = cache.double()
        again = _to_codes(old * scale.double()[:, :, None, None] / now.double()[:, :, None, None], kind)
        early = torch.arange(block, device=page.device)[None, None, :, None] < kept[:, None, None, None]
        cache.copy_(torch.where(grown[:, :, None, None] & early, again.double(), old))
        codes = _to_codes(x / now.double()[page][:, :, None], kind)
        cache.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
        scale.copy_(torch.where(touched[:, None], now, scale))
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def _plain_attend(s):
    case = s["case"]
    block, heads, dim = case["block"], case["heads"], case["dim"]
    group = case["q_heads"] // heads
    width = -(-s["max_len"] // block)
    batch, longest, tokens = case["batch"], s["max_new"], s["q"].shape[0]
    table = s["table"][:, :width].long()

    def dense(name):
        cache = s[name + "_cache"]
        x = cache.view(torch.uint8)[table].view(cache.dtype).float() * s[name + "_scale"][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, heads, width * block, dim)

    new = s["query_start"][1:] - s["query_start"][:-1]
    q = torch.zeros(batch, longest, case["q_heads"], dim, device=table.device)
    q[s["owner"], s["place"]] = s["q"].float()
    q = q.reshape(batch, longest, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * longest, dim)
    scores = (q @ dense("k").transpose(2, 3)).reshape(batch, heads, group, longest, -1) * (1.0 / math.sqrt(dim))
    last = (s["seq_lens"] - new)[:, None] + torch.arange(longest, device=table.device)  # position of every query
    seen = torch.arange(width * block, device=table.device)[None, None, :] <= last[:, :, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - most.masked_fill(most == -math.inf, 0.0))
    total = p.sum(dim=-1, keepdim=True)
    o = p.reshape(batch, heads, group * longest, -1) @ dense("v")
    o = o.reshape(batch, heads, group, longest, dim) / total.masked_fill(total == 0, 1.0)
    lse = (most + torch.log(total)).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, longest, case["q_heads"], dim)[s["owner"], s["place"]]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, longest, case["q_heads"])[s["owner"], s["place"]]
    return [o.to(s["q"].dtype), lse]


# ----------------------------------------------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "linear":
        n, k, t = case["rows"], case["cols"], case["tokens"]
        groups = 1 if case["group"] == -1 else k // case["group"]
        per = 1 if case["codec"] == "nvfp4" else 2 + (1 if case["zp"] else 0)
        return {"bytes": n * -(-k // 8) * 4 + n * groups * per + 2 * t * (n + k) + (2 * n if case["bias"] else 0), "flops": 2 * t * n * k}
    lens, heads, dim, block = _lens(case), case["heads"], case["dim"], case["block"]
    new = sum(m for _, m in lens)
    if case["op"] == "append":
        blocks = sum(-(-t // block) - (t - m) // block for t, m in lens)
        return {"bytes": 2 * new * heads * dim * 3 + 2 * blocks * heads * 4, "flops": 4 * new * heads * dim}
    held = sum(t for t, _ in lens)
    pairs = sum(m * (t - m) + m * (m + 1) // 2 for t, m in lens if t >= m)
    return {"bytes": 2 * held * heads * dim + 2 * sum(-(-t // block) for t, _ in lens) * heads * 4 + new * case["q_heads"] * (4 * dim + 4),
            "flops": 4 * pairs * case["q_heads"] * dim}


# ---------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)


def _exact_linear(case, s):
    n, k, size = case["rows"], case["cols"], s["group"]
    x = s["x"].double()
    out = torch.empty(case["tokens"], n, dtype=torch.float64, device="cuda")
    raw = s["q"].view(torch.uint8) if case["codec"] == "nvfp4" else s["q"].contiguous().view(torch.uint8)
    for i in range(0, n, 1024):  # byte j of a row holds columns 2j (low half) and 2j + 1
        b = raw[i:i + 1024].long()
        c = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.float64, device="cuda")
        if case["codec"] == "int4":
            c[:, 0::2], c[:, 1::2] = b % 16 - 8, b // 16 - 8
        else:
            values = torch.tensor(E2M1 + tuple(-e for e in E2M1), dtype=torch.float64, device="cuda")
            c[:, 0::2], c[:, 1::2] = values[b % 16], values[b // 16]
        c = c[:, :k]
        scale = s["scale"][i:i + 1024].double().repeat_interleave(size, dim=1)
        if s["zp"] is not None:
            c = c - s["zp"][i:i + 1024].double().repeat_interleave(size, dim=1)
        if s["gs"] is not None:
            scale = scale / s["gs"].double()
        out[:, i:i + 1024] = x @ (c * scale).t()
    if s["bias"] is not None:
        out += s["bias"].double()
    return out


def _nearest(x, kind):
    """The code value nearest to each number: from the list of all code values, ties to the even one."""
    if kind == "int8":
        grid = torch.arange(-128, 128, dtype=torch.float64, device=x.device)
        even = torch.arange(-128, 128, device=x.device) % 2 == 0
    else:
        up = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
        up = torch.tensor(up[:127], dtype=torch.float64, device=x.device)  # the last pattern is not a number
        grid = torch.cat((-up[1:].flip(0), up))
        even = torch.cat((torch.arange(1, 127, device=x.device).flip(0), torch.arange(127, device=x.device))) % 2 == 0
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    down, above = x - grid[lo], grid[hi] - x
    return torch.where((above < down) | ((above == down) & even[hi]), grid[hi], grid[lo])


def _exact_append(case, s):
    block, kind = case["block"], case["cache"]
    table, out = s["table"].tolist(), []
    lens = _lens(case)
    for name in ("k", "v"):
        cache, scale, x = s[name + "_cache"].double(), s[name + "_scale"].double(), s[name].double()
        at = 0
        for b, (total, new) in enumerate(lens):
            first = total - new
            while first < total:
                page, begin = table[b][first // block], first % block
                end = min(block, begin + total - first)
                rows = x[at:at + end - begin]  # [tokens, heads, dim]
                now = (rows.abs().amax(dim=(0, 2)) / HALF_RANGE[kind]).float().double().clamp(min=EPS)  # a scale is held in 32 bits
                if begin:
                    grown = torch.maximum(scale[page], now)
                    kept = _nearest(cache[page, :, :begin] * (scale[page] / grown)[:, None, None], kind)
                    cache[page, :, :begin] = torch.where((grown > scale[page])[:, None, None], kept, cache[page, :, :begin])
                    now = grown
                scale[page] = now
                cache[page, :, begin:end] = _nearest((rows / now[None, :, None]).transpose(0, 1), kind)
                at += end - begin
                first += end - begin
        out += [cache if kind == "e4m3" else cache.to(torch.int8), scale]
    return [out[0], out[2], out[1], out[3]]


def _exact_attend(case, s):
    block, heads, dim = case["block"], case["heads"], case["dim"]
    group = case["q_heads"] // heads
    outs, lses, at = [], [], 0
    for b, (total, new) in enumerate(_lens(case)):
        pages = s["table"][b, :-(-total // block)].long()
        q = s["q"][at:at + new].double().reshape(new, heads, group, dim)
        at += new

        def rows(name):
            cache = s[name + "_cache"]
            x = cache.view(torch.uint8)[pages].view(cache.dtype).double() * s[name + "_scale"][pages].double()[:, :, None, None]
            return x.transpose(1, 2).reshape(-1, heads, dim)[:total]

        k, v = rows("k"), rows("v")
        score = torch.einsum("ihgd,jhd->hgij", q, k) / math.sqrt(dim)
        i = torch.arange(new, device="cuda")[:, None] + (total - new)
        score = torch.where(torch.arange(total, device="cuda")[None, :] <= i, score, -math.inf)
        lse = torch.logsumexp(score, dim=-1) if total else torch.full((heads, group, new), -math.inf, dtype=torch.float64, device="cuda")
        weight = torch.exp(score - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        outs.append(torch.einsum("hgij,jhd->ihgd", weight, v).reshape(new, heads * group, dim))
        lses.append(lse.permute(2, 0, 1).reshape(new, heads * group))
    return [torch.cat(outs), torch.cat(lses)]
