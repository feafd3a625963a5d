"""The operators that serve a compressed model, against the same formulas in 64 bits.

Tolerances, fixed before the first run.  A result is rounded once (half a step of its type, relative).  In front of that
there are fp32 sums: a chain of n additions is off by at most n * 2^-23 of the sum of magnitudes (2^-23, not 2^-24, since
tensor cores may cut instead of rounding).  The attention may hold its weights in float16 (2^-11 relative, 2^-25 absolute
below the normal range) and its queries in float16 scaled to the row's maximum (2^-25 of that maximum)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # finfo.eps / 2
E2M1 = [0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------- the 4-bit product

def make_linear(tokens, rows, cols, codec, group, zp, bias, dtype, scale_dtype, seed=0):
    g = gen(seed)
    group = cols if group == -1 else group
    s = dict(x=torch.randn(tokens, cols, generator=g, device="cuda").to(dtype), zp=None, gs=None, bias=None, codec=codec, group=group)
    if codec == "pack32":
        codes = torch.randint(0, 16, (rows, -(-cols // 8) * 8), generator=g, device="cuda", dtype=torch.int32)  # random bits behind the last column too
        s["q"] = (codes.reshape(rows, codes.shape[1] // 8, 8) << torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)).sum(-1).to(torch.int32)
        s["codes"] = codes[:, :cols].double() - 8
        s["scale"] = (torch.rand(rows, cols // group, generator=g, device="cuda") * 0.1 + 0.001).to(scale_dtype)
        if zp:
            s["zp"] = torch.randint(-8, 8, (rows, cols // group), generator=g, device="cuda", dtype=torch.int8)
    else:
        s["q"] = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
        both = torch.stack((s["q"] & 15, s["q"] >> 4), -1).reshape(rows, cols).long()
        s["codes"] = torch.tensor(E2M1, dtype=torch.float64, device="cuda")[both]
        s["scale"] = (torch.randn(rows, cols // group, generator=g, device="cuda") * 100).clamp(-448, 448).to(scale_dtype)
        s["gs"] = torch.tensor([331.7], device="cuda")
    if bias:
        s["bias"] = torch.randn(rows, generator=g, device="cuda").to(dtype)
    return s


def call_linear(s, x=None, **kw):
    from compressed_tensors_b200 import torch_ops as ops

    a = dict(qtype=ops.QINT if s["codec"] == "pack32" else ops.QFLOAT, col_group=s["group"], scale_row_stride=s["scale"].shape[1], codec=s["codec"],
             global_scale=s["gs"], bias=s["bias"])
    return ops.dequantize_linear(s["x"] if x is None else x, s["q"], s["scale"], s["zp"], **{**a, **kw})


def check_linear(s, got, x=None):
    x = s["x"] if x is None else x
    scale = s["scale"].double()
    if s["gs"] is not None:
        scale = scale / s["gs"].double()
    codes = s["codes"]
    if s["zp"] is not None:
        codes = codes - s["zp"].double().repeat_interleave(s["group"], 1)
    w = codes * scale.repeat_interleave(s["group"], 1)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if s["bias"] is not None:
        want, size = want + s["bias"].double(), size + s["bias"].double().abs()
    tol = HALF[x.dtype] * want.abs() + (x.shape[-1] / 16 + 64) * 2.0 ** -23 * size * 1.01 + 2.0 ** -25
    assert got.dtype == x.dtype and got.shape == want.shape
    off = ((got.double() - want).abs() - tol).max() if want.numel() else torch.zeros(())
    assert float(off) <= 0, f"outside the tolerance by {float(off):.3g}"


@pytest.mark.parametrize("codec, group, zp", [("pack32", 128, False), ("pack32", 128, True), ("pack32", 64, False), ("pack32", 32, True), ("pack32", -1, False),
                                              ("pack32", -1, True), ("fp4x2", 16, False), ("fp4x2", 32, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens, rows, cols", [(1, 128, 128), (1, 1000, 2048), (3, 17, 4096), (8, 129, 1664), (9, 256, 384), (16, 1, 256), (31, 200, 640), (33, 144, 256),
                                                (70, 96, 512), (10, 8200, 256), (24, 8192, 512)])
def test_linear(tokens, rows, cols, codec, group, zp, dtype):
    s = make_linear(tokens, rows, cols, codec, group, zp, tokens % 2 == 1, dtype, torch.float8_e4m3fn if codec == "fp4x2" else dtype, seed=tokens)
    check_linear(s, call_linear(s))


@pytest.mark.parametrize("cols, codec, group", [(8, "pack32", 8), (1, "pack32", 1), (17, "pack32", 17), (1001, "pack32", 7), (96, "pack32", 24), (96, "pack32", 96), (160, "pack32", 32),
                                                (4104, "pack32", -1), (48, "pack32", 16), (2, "fp4x2", 2), (16, "fp4x2", 16), (48, "fp4x2", 16), (80, "fp4x2", 16),
                                                (24, "fp4x2", 8), (1040, "fp4x2", 16), (96, "fp4x2", 32)])
@pytest.mark.parametrize("tokens", [1, 5, 12])
def test_linear_odd_columns(cols, codec, group, tokens):
    for rows in (1, 37):
        s = make_linear(tokens, rows, cols, codec, group, codec == "pack32" and tokens == 5, False, torch.bfloat16,
                        torch.float8_e4m3fn if codec == "fp4x2" else torch.bfloat16, seed=cols)
        check_linear(s, call_linear(s))


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("codec", ["pack32", "fp4x2"])
def test_linear_scale_types(codec, scale_dtype):
    s = make_linear(4, 100, 256, codec, 32 if codec == "pack32" else 16, False, False, torch.bfloat16, scale_dtype)
    check_linear(s, call_linear(s))


def test_linear_empty_and_shapes():
    s = make_linear(6, 40, 256, "pack32", 128, False, True, torch.bfloat16, torch.bfloat16)
    check_linear(s, call_linear(s, x=s["x"].reshape(2, 3, 256)).reshape(6, 40))
    assert tuple(call_linear(s, x=s["x"][0]).shape) == (40,)
    assert tuple(call_linear(s, x=s["x"][:0]).shape) == (0, 40)
    wide = torch.randn(6, 512, generator=gen(1), device="cuda").to(torch.bfloat16)
    check_linear(s, call_linear(s, x=wide[:, 128:384]), wide[:, 128:384])  # strided rows
    check_linear(s, call_linear(s, x=wide.flatten()[1:1 + 6 * 256].view(6, 256)), wide.flatten()[1:1 + 6 * 256].view(6, 256))  # off the 16-byte grid
    padded = torch.zeros(40 * 32 + 1, dtype=torch.int32, device="cuda")
    padded[1:] = s["q"].flatten()
    check_linear({**s, "q": padded[1:].view(40, 32)}, call_linear({**s, "q": padded[1:].view(40, 32)}))  # words off the 16-byte grid
    one = make_linear(3, 40, 256, "pack32", -1, False, False, torch.bfloat16, torch.bfloat16)
    one["scale"] = one["scale"][:1].expand(40, 1)  # one scale for the whole tensor
    check_linear(one, call_linear({**one, "scale": one["scale"][:1]}, scale_row_stride=0))
    none = make_linear(3, 0, 256, "pack32", 128, False, False, torch.bfloat16, torch.bfloat16)
    assert tuple(call_linear(none).shape) == (3, 0)


@pytest.mark.parametrize("codec", ["pack32", "fp4x2"])
def test_linear_values_at_the_edges(codec):
    """Infinities and NaN stay in their token, large and tiny numbers keep their range."""
    s = make_linear(5, 64, 512, codec, 128 if codec == "pack32" else 16, False, False, torch.bfloat16,
                    torch.bfloat16 if codec == "pack32" else torch.float8_e4m3fn)
    x = s["x"].clone()
    x[1, 3], x[2, 70] = float("nan"), float("inf")
    x[3] *= 2.0 ** 100
    x[4] *= 2.0 ** -100
    got = call_linear(s, x=x)
    clean = torch.tensor([0, 3, 4], device="cuda")
    keep = dict(s, x=x[clean])
    w = s["codes"] * (s["scale"].double() / (1 if s["gs"] is None else s["gs"].double())).repeat_interleave(s["group"], 1)
    want = keep["x"].double() @ w.t()
    size = keep["x"].double().abs() @ w.abs().t()
    assert bool(((got[clean].double() - want).abs() <= HALF[x.dtype] * want.abs() + 96 * 2.0 ** -23 * size * 1.01).all())
    assert bool(got[1].isnan().all()) and not bool(got[2].isfinite().any())


# --------------------------------------------------------------------------------------------------------- the cache

def make_cache(lens, heads, dim, block, cdtype, seed=0, layout="hnd", spare=2, scale_spread=1.0):
    """Random codes and scales, pages in random order; what no request owns holds codes and scales that would show."""
    g = gen(seed)
    used = [-(-max(n, 0) // block) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = max(used + [1]) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
        at += u
    c = dict(block_table=table.cuda(), seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for n in ("k", "v"):
        x = torch.randn(pages, heads, block, dim, generator=g, device="cuda") * (60 if cdtype is torch.float8_e4m3fn else 30)
        x = x.clamp(-448, 448).to(cdtype) if cdtype is torch.float8_e4m3fn else x.round().clamp(-128, 127).to(cdtype)
        if layout == "nhd":
            x = x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(cdtype)
        c[n + "_cache"] = x
        c[n + "_scale"] = torch.exp(torch.randn(pages, heads, generator=g, device="cuda") * scale_spread) * 0.02
    return c


def starts(rows, extra=0):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda"), out[-1] + extra


def call_attention(c, q, qs, **kw):
    from compressed_tensors_b200 import torch_ops as ops

    return ops.kv_cache_attention(q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["seq_lens"], qs, return_lse=True, **kw)


def dense(c, name, b, n, block):
    codes, scale = c[name + "_cache"].double(), c[name + "_scale"].double()
    pages = c["block_table"][b, :-(-n // block)].long()
    ok = (pages >= 0) & (pages < codes.shape[0])
    x = codes[pages.clamp(0, codes.shape[0] - 1)] * scale[pages.clamp(0, codes.shape[0] - 1)][:, :, None, None]
    heads, dim = codes.shape[1], codes.shape[3]
    return x.transpose(1, 2).reshape(-1, heads, dim)[:n], ok.repeat_interleave(block)[:n], scale[pages.clamp(0, codes.shape[0] - 1)].repeat_interleave(block, 0)[:n]


def check_attention(c, q, qs, got, lse, causal=True, scale=None):
    heads, block, dim = c["k_cache"].shape[1:]
    group = q.shape[1] // heads
    scale = dim ** -0.5 if scale is None else scale
    assert got.shape == q.shape and got.dtype == q.dtype and lse.shape == q.shape[:2] and lse.dtype == torch.float32
    seen = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    most_code = 448.0 if c["v_cache"].dtype is torch.float8_e4m3fn else 128.0
    for b, (lo, hi) in enumerate(zip(qs.tolist()[:-1], qs.tolist()[1:])):
        length = max(int(c["seq_lens"][b]), 0)
        n = min(length, c["block_table"].shape[1] * block)
        rows = hi - lo
        if rows == 0:
            continue
        seen[lo:hi] = True
        x = q[lo:hi].double().reshape(rows, heads, group, dim)
        k, ok, _ = dense(c, "k", b, n, block)
        v, _, vs = dense(c, "v", b, n, block)
        i = torch.arange(rows, device="cuda")[:, None] + (length - rows)
        j = torch.arange(n, device="cuda")[None, :]
        visible = ((j <= i) if causal else torch.ones_like(j <= i)) & ok[None, :]
        s = torch.einsum("ihgd,jhd->hgij", x, k) * scale
        size = torch.einsum("ihgd,jhd->hgij", x.abs(), k.abs()) * abs(scale)
        qmax = x.abs().amax(-1).permute(1, 2, 0)  # heads, group, rows
        ksum = k.abs().sum(-1).t()[:, None, None, :] if n else torch.zeros(heads, 1, 1, 0, device="cuda", dtype=torch.float64)
        ds = (dim / 16 + 24) * 2.0 ** -23 * size + 2.0 ** -25 * qmax[..., None] * ksum * abs(scale) + 2.0 ** -22 * s.abs()
        ds = ds.masked_fill(~visible, 0).amax(-1) if n else torch.zeros(heads, group, rows, device="cuda", dtype=torch.float64)
        s = s.masked_fill(~visible, -math.inf)
        want_lse = torch.logsumexp(s, -1) if n else torch.full((heads, group, rows), -math.inf, device="cuda", dtype=torch.float64)
        p = torch.exp(s - want_lse.masked_fill(want_lse == -math.inf, 0)[..., None])
        want = torch.einsum("hgij,jhd->ihgd", p, v).reshape(rows, -1, dim)
        mag = torch.einsum("hgij,jhd->ihgd", p, v.abs()).reshape(rows, -1, dim)
        chain = (n / 16 + 64) * 2.0 ** -23
        top = (p * vs.t()[:, None, None, :]).amax(-1) if n else torch.zeros_like(want_lse)
        under = (n * 2.0 ** -25 * most_code * top).permute(2, 0, 1).reshape(rows, -1)[..., None]
        dsr = ds.permute(2, 0, 1).reshape(rows, -1)
        tol = HALF[q.dtype] * want.abs() + (2.0 ** -11 + 2 * dsr[..., None] + chain) * 1.02 * mag + under + 2.0 ** -25 * (q.dtype is torch.float16)
        g = got[lo:hi].double()
        assert bool(((g - want).abs() <= tol).all()), f"request {b}: {float(((g - want).abs() - tol).max()):.3g} outside the tolerance"
        wl, gl = want_lse.permute(2, 0, 1).reshape(rows, -1), lse[lo:hi].double()
        empty = wl == -math.inf
        assert torch.equal(gl == -math.inf, empty) and bool((g[empty] == 0).all())
        assert bool(((gl - wl).masked_fill(empty, 0).abs() <= (dsr + chain + 2.0 ** -22 * (1 + wl.masked_fill(empty, 0).abs())) * 1.02).all())
    assert bool((got[~seen] == 0).all()) and bool((lse[~seen] == -math.inf).all())


ROWS = [  # (cached tokens, query rows) per request
    [(1, 1)], [(0, 1)], [(0, 0), (7, 1), (0, 0)], [(200, 1)], [(15, 1), (16, 1), (17, 1), (31, 1), (33, 1), (64, 1), (65, 1)],
    [(1000, 1), (3, 1), (0, 1), (257, 1)], [(5, 5)], [(40, 3), (2, 2), (100, 9)], [(300, 130), (64, 1), (129, 129)], [(3, 5), (0, 4)], [(2500, 1)],
    [(700, 40), (1, 1), (90, 0), (513, 257)],
]


@pytest.mark.parametrize("shape", ROWS, ids=str)
@pytest.mark.parametrize("cdtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("heads, group, dim, block, dtype", [(2, 4, 128, 64, torch.bfloat16), (1, 1, 64, 16, torch.float16), (2, 7, 128, 32, torch.float16), (1, 16, 256, 16, torch.bfloat16),
                                                             (3, 8, 64, 128, torch.bfloat16), (1, 3, 80, 16, torch.bfloat16), (2, 2, 33, 5, torch.float16), (1, 40, 128, 48, torch.bfloat16)])
def test_attention(shape, heads, group, dim, block, dtype, cdtype):
    c = make_cache([n for n, _ in shape], heads, dim, block, cdtype, seed=len(shape))
    qs, tokens = starts([m for _, m in shape], extra=2)
    q = torch.randn(tokens, heads * group, dim, generator=gen(7), device="cuda").to(dtype)
    for causal in (True, False):
        check_attention(c, q, qs, *call_attention(c, q, qs, causal=causal), causal=causal)


@pytest.mark.parametrize("rows", [1, 60])
def test_attention_strides_and_layouts(rows):
    """Heads behind tokens in the cache, queries as a slice of a fused projection, a table that is a slice of a wider one."""
    for offset in (0, 8, 1):
        c = make_cache([333, 90], 2, 128, 32, torch.float8_e4m3fn, layout="nhd")
        wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
        wide[:, 3:3 + c["block_table"].shape[1]] = c["block_table"]
        c["block_table"] = wide[:, 3:3 + c["block_table"].shape[1]]
        qs, tokens = starts([rows, rows])
        fused = torch.randn(tokens, 13 * 128, generator=gen(3), device="cuda").to(torch.bfloat16)
        q = fused[:, offset:offset + 8 * 128].unflatten(1, (8, 128))
        check_attention(c, q, qs, *call_attention(c, q, qs))
        t = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
        check_attention(c, t, qs, *call_attention(c, t, qs, softmax_scale=0.3), scale=0.3)
    pool = torch.zeros(2 * c["k_cache"].numel() + 1, dtype=torch.uint8, device="cuda")  # codes off the 16-byte grid
    odd = pool[1:1 + c["k_cache"].numel()].view(c["k_cache"].dtype).view(c["k_cache"].shape)
    odd.copy_(c["k_cache"])
    check_attention({**c, "k_cache": odd}, q, qs, *call_attention({**c, "k_cache": odd}, q, qs))


@pytest.mark.parametrize("dim", [128, 80])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_wild_tables_and_lengths(rows, dim):
    """Block numbers outside the cache, lengths beyond the table or below zero: those tokens are left out."""
    c = make_cache([200, 150, 90, 64], 2, dim, 16, torch.int8)
    c["block_table"][0, 3], c["block_table"][1, 0] = -5, 2 ** 31 - 1
    c["block_table"][1, 4] = c["k_cache"].shape[0]
    c["seq_lens"] = torch.tensor([200, 150, -3, 10 ** 9], dtype=torch.int32, device="cuda")
    qs, tokens = starts([rows] * 4)
    q = torch.randn(tokens, 4, dim, generator=gen(5), device="cuda").to(torch.bfloat16)
    for causal in (True, False):
        check_attention(c, q, qs, *call_attention(c, q, qs, causal=causal), causal=causal)


@pytest.mark.parametrize("dim, dtype", [(128, torch.bfloat16), (64, torch.float16), (96, torch.bfloat16)])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_extreme_scales(rows, dim, dtype):
    """Value scales of very different size from block to block, all-zero blocks with a zero scale, scores far apart."""
    c = make_cache([700, 333], 2, dim, 16, torch.float8_e4m3fn, scale_spread=4.0, seed=9)
    c["v_scale"][::5] = 0.0
    c["k_scale"][1::3] *= 50
    qs, tokens = starts([rows, rows])
    q = (torch.randn(tokens, 8, dim, generator=gen(5), device="cuda") * 3).to(dtype)
    check_attention(c, q, qs, *call_attention(c, q, qs))
    big = q * 2.0 ** (60 if dtype is torch.bfloat16 else 6)  # one key takes all the weight
    small = dict(c, k_scale=c["k_scale"] * 2.0 ** (-60 if dtype is torch.bfloat16 else -6))
    check_attention(small, big, qs, *call_attention(small, big, qs))


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_not_a_number(rows):
    """A NaN in a query, a key scale or a value scale reaches the queries that see it and no others."""
    for what in ("q", "k_scale", "v_scale"):
        c = make_cache([300, 200], 2, 128, 16, torch.float8_e4m3fn)
        qs, tokens = starts([rows, rows])
        q = torch.randn(tokens, 4, 128, generator=gen(5), device="cuda").to(torch.bfloat16)
        hit = torch.zeros(tokens, 4, dtype=torch.bool, device="cuda")
        if what == "q":
            q[rows - 1, 1, 5] = float("nan")
            hit[rows - 1, 1] = True
        else:
            c[what][int(c["block_table"][1, 2]), 0] = float("nan")
            hit[rows:, :2] = True
        out, _ = call_attention(c, q, qs)
        assert torch.equal(out.isnan().all(-1), hit) and torch.equal(out.isnan().any(-1), hit)


# ------------------------------------------------------------------------------------------------------------ append

def nearest(x, cdtype):
    """Correctly rounded codes of 64-bit numbers, ties to even."""
    if cdtype is torch.int8:
        return x.round().clamp(-128, 127)
    _, e = torch.frexp(x)
    step = (((e - 1).clamp(min=-6) - 3).long() + 1023 << 52).view(torch.float64)  # a power of two, exact
    return ((x / step).round() * step).clamp(-448, 448)


def append_reference(c, k, v, qs):
    out = {n: c[n].clone() for n in ("k_scale", "v_scale")}
    heads, block, dim = c["k_cache"].shape[1:]
    half = 448.0 if c["k_cache"].dtype is torch.float8_e4m3fn else 127.5
    for name, x in (("k", k), ("v", v)):
        codes = c[name + "_cache"].double()
        scale = out[name + "_scale"]
        for b, (lo, hi) in enumerate(zip(qs.tolist()[:-1], qs.tolist()[1:])):
            total = int(c["seq_lens"][b])
            p = total - (hi - lo)
            while p < total:
                j = p // block
                end = min(total, (j + 1) * block)
                if p < 0:
                    p = min(0, end)
                    continue
                page = int(c["block_table"][b, j]) if j < c["block_table"].shape[1] else -1
                if 0 <= page < codes.shape[0]:
                    rows = x[hi - (total - p):hi - (total - end)].double()
                    now = (rows.abs().amax(dim=(0, 2)) / half).float().clamp(min=2.0 ** -23)
                    kept = p - j * block
                    if kept:
                        now = torch.maximum(scale[page], now)
                        again = nearest(codes[page, :, :kept] * scale[page].double()[:, None, None] / now.double()[:, None, None], c["k_cache"].dtype)
                        codes[page, :, :kept] = torch.where((now > scale[page])[:, None, None], again, codes[page, :, :kept])
                    codes[page, :, kept:kept + end - p] = nearest(rows.transpose(0, 1) / now.double()[:, None, None], c["k_cache"].dtype)
                    scale[page] = now
                p = end
        out[name + "_cache"] = codes
    return out


def check_append(c, k, v, qs):
    from compressed_tensors_b200 import torch_ops as ops

    want = append_reference(c, k, v, qs)
    args = (k, v, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["seq_lens"], qs)
    ops.kv_cache_append(*args)
    for n, w in want.items():
        assert torch.equal(c[n].double(), w.double()), n
    before = {n: c[n].clone() for n in want}
    ops.kv_cache_append(*args)  # the same rows again change nothing
    for n, w in before.items():
        assert torch.equal(c[n].view(torch.uint8), w.view(torch.uint8)), n


@pytest.mark.parametrize("cdtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, dim, block, layout", [(2, 128, 64, "hnd"), (1, 64, 16, "nhd"), (3, 256, 32, "hnd"), (2, 80, 16, "nhd"), (2, 33, 5, "hnd"), (1, 128, 256, "hnd")])
@pytest.mark.parametrize("shape", [[(1, 1)], [(0, 0), (64, 1), (65, 1), (17, 1)], [(200, 130), (3, 3), (90, 0), (1, 1), (129, 2)], [(16, 16), (2000, 700)], [(5, 9), (0, 3)]], ids=str)
def test_append(shape, heads, dim, block, layout, dtype, cdtype):
    c = make_cache([n for n, _ in shape], heads, dim, block, cdtype, layout=layout)
    qs, tokens = starts([m for _, m in shape], extra=2)
    fused = torch.randn(tokens, heads * 3, dim, generator=gen(2), device="cuda").to(dtype)
    fused *= torch.exp(2 * torch.randn(tokens, heads * 3, 1, generator=gen(3), device="cuda")).to(dtype)  # some blocks grow, some do not
    check_append(c, fused[:, heads:2 * heads], fused[:, 2 * heads:], qs)


def test_append_zero_tiny_and_wild():
    """All-zero rows take the smallest scale; unaligned rows; pages outside the cache are left alone."""
    for offset in (0, 3):
        c = make_cache([40, 50, 33], 2, 128, 16, torch.float8_e4m3fn)
        c["block_table"][1, 1], c["block_table"][2, 0] = -1, 10 ** 6
        qs, tokens = starts([20, 50, 33])
        k = torch.randn(tokens * 2 * 128 + offset, generator=gen(2), device="cuda").to(torch.bfloat16)[offset:].view(tokens, 2, 128)
        k[:20] = 0
        check_append(c, k, k * 2.0 ** -80, qs)


def test_append_not_a_number():
    from compressed_tensors_b200 import torch_ops as ops

    c = make_cache([40, 20], 2, 64, 16, torch.float8_e4m3fn)
    qs, _ = starts([1, 20])
    k = torch.randn(21, 2, 64, generator=gen(2), device="cuda").to(torch.bfloat16)
    k[3, 1, 7] = float("nan")
    ops.kv_cache_append(k, k, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["seq_lens"], qs)
    bad = torch.zeros_like(c["k_scale"], dtype=torch.bool)
    bad[int(c["block_table"][1, 0]), 1] = True
    assert torch.equal(c["k_scale"].isnan(), bad) and torch.equal(c["v_scale"].isnan(), bad)


# ------------------------------------------------------------------------------------- together, graphs, other streams

def decode_state(seed=0):
    """A small decoder layer's attention: packed projections around an 8-bit cache."""
    g = gen(seed)
    heads, q_heads, dim, hidden, block = 2, 8, 64, 512, 16
    lens = [70, 5, 129]
    c = make_cache([n + 8 for n in lens], heads, dim, block, torch.int8, seed=seed)
    c["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = make_linear(3, (q_heads + 2 * heads) * dim, hidden, "pack32", 128, False, False, torch.bfloat16, torch.bfloat16, seed + 1)
    o = make_linear(3, hidden, q_heads * dim, "fp4x2", 16, False, False, torch.bfloat16, torch.float8_e4m3fn, seed + 2)
    qkv["scale"] *= 0.1
    x = torch.randn(3, hidden, generator=g, device="cuda").to(torch.bfloat16)
    qs, _ = starts([1, 1, 1])
    return c, qkv, o, x, qs, (q_heads, heads, dim)


def decode_step(state):
    from compressed_tensors_b200 import torch_ops as ops

    c, qkv, o, x, qs, (q_heads, heads, dim) = state
    y = call_linear(qkv, x=x).unflatten(1, (q_heads + 2 * heads, dim))
    ops.kv_cache_append(y[:, q_heads:q_heads + heads], y[:, q_heads + heads:], c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"],
                        c["block_table"], c["seq_lens"], qs)
    att, lse = call_attention(c, y[:, :q_heads], qs)
    return y, att, lse, call_linear(o, x=att.flatten(1))


@pytest.mark.parametrize("fmt, kw", [("pack-quantized", dict(num_bits=4, symmetric=True, strategy="group", group_size=128)),
                                     ("pack-quantized", dict(num_bits=4, symmetric=False, strategy="group", group_size=32)),
                                     ("pack-quantized", dict(num_bits=4, symmetric=True, strategy="channel")),
                                     ("nvfp4-pack-quantized", dict(num_bits=4, type="float", symmetric=True, strategy="tensor_group", group_size=16))])
def test_compressed_linear_keeps_its_packed_weight(fmt, kw):
    from compressed_tensors_b200 import _lib as L
    from compressed_tensors_b200.compressors import ModelCompressor
    from compressed_tensors_b200.linear import CompressedLinear
    from compressed_tensors_b200.quantization import (QuantizationArgs, QuantizationConfig, QuantizationScheme, QuantizationStatus, apply_quantization_config,
                                                      calibrate_weight_qparams)

    torch.manual_seed(3)
    model = torch.nn.Sequential(torch.nn.Linear(384, 200, bias=True)).to(torch.bfloat16).cuda()
    scheme = QuantizationScheme(targets=["Linear"], weights=QuantizationArgs(**kw))
    cfg = QuantizationConfig(config_groups={"g": scheme}, format=fmt)
    apply_quantization_config(model, cfg)
    calibrate_weight_qparams(model[0])
    bias = model[0].bias.data.clone()
    sd = ModelCompressor(quantization_config=cfg).compress(model)
    mods = []
    for keep in (True, False):
        lin = torch.nn.Linear(384, 200, bias=True, dtype=torch.bfloat16).cuda()
        mod = CompressedLinear.from_linear(lin, scheme, fmt, keep_packed=keep)
        _, unexpected = mod.load_state_dict({k.removeprefix("0."): v for k, v in sd.items() if k.startswith("0.")}, strict=False)
        assert not unexpected
        mods.append(mod)
    packed, dense = mods
    weight = dense.compressor.decompress_module(dense).double()
    with torch.no_grad():
        for tokens in (1, 7, 32):
            x = torch.randn(tokens, 384, dtype=torch.bfloat16, device="cuda")
            assert packed.packed_product(x) is not None
            y = packed(x)
            want, size = x.double() @ weight.t() + bias.double(), x.double().abs() @ weight.abs().t() + bias.double().abs()
            # the dense weight is rounded to bf16 (half a step each), the packed product does not round it
            assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 96 * 2.0 ** -23) * size).all())
            assert packed.quantization_status == QuantizationStatus.COMPRESSED and not hasattr(packed, "weight")
        many = torch.randn(33, 384, dtype=torch.bfloat16, device="cuda")
        assert packed.packed_product(many) is None and packed.packed_product(many[:2].float()) is None
        assert torch.equal(packed(many), dense(many))
    few = torch.randn(3, 384, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    assert packed.packed_product(few) is None  # a gradient is wanted: the dense way gives it
    packed(few).sum().backward()
    assert bool(((few.grad[0].double() - weight.sum(0)).abs() <= 2.0 ** -8 * weight.sum(0).abs() + 200 * 2.0 ** -23 * weight.abs().sum(0)).all())
    assert L.launch_count() > 0


def test_a_decoding_step():
    state = decode_state()
    c, qkv, o, x, qs, (q_heads, heads, dim) = state
    before = {n: t.clone() for n, t in c.items()}
    for _ in range(5):
        y, att, lse, out = decode_step(state)
        check_linear(qkv, y.flatten(1), x)
        want = append_reference(before, y[:, q_heads:q_heads + heads], y[:, q_heads + heads:], qs)
        for n, w in want.items():
            assert torch.equal(c[n].double(), w.double()), n
        check_attention(c, y[:, :q_heads], qs, att, lse)
        check_linear(o, out, att.flatten(1))
        c["seq_lens"] += 1
        x = state[3].copy_(out)
        before = {n: t.clone() for n, t in c.items()}


def test_captured_steps_share_nothing():
    """Two captured graphs and an eager call in turn, each with lengths that grow between replays."""
    a, b = decode_state(1), decode_state(2)
    eager = [decode_state(1), decode_state(2)]
    graphs = []
    for s in (a, b):
        keep = {n: t.clone() for n, t in s[0].items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_step(s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode_step(s)
        for n, t in keep.items():  # the warm-up appended: start again
            s[0][n].view(torch.uint8).copy_(t.view(torch.uint8))
        graphs.append((g, out))
    for step in range(3):
        for i in (0, 1):
            graphs[i][0].replay()
            want = decode_step(eager[i])
            for got, w in zip(graphs[i][1], want):
                assert torch.equal(got, w)
            for s in ((a, b)[i], eager[i]):
                s[0]["seq_lens"] += 1


@pytest.mark.parametrize("rows", [1, 40])
def test_a_captured_attention_follows_its_lengths(rows):
    """Requests long enough to be cut into pieces that a second kernel joins; lengths and queries change between replays."""
    c = make_cache([6000, 700, 40], 2, 128, 64, torch.float8_e4m3fn)
    c["seq_lens"] = torch.tensor([100, 60, 40], dtype=torch.int32, device="cuda")
    qs, tokens = starts([rows] * 3, extra=1)
    q = torch.randn(tokens, 8, 128, generator=gen(1), device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call_attention(c, q, qs)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call_attention(c, q, qs)
    for i, lens in enumerate(([100, 60, 40], [6000, 700, 40], [0, 1, 0], [5990, 0, 33])):
        c["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn(tokens, 8, 128, generator=gen(i), device="cuda").to(torch.bfloat16))
        g.replay()
        check_attention(c, q, qs, *out)
        eager = call_attention(c, q, qs)
        assert torch.equal(eager[0], out[0]) and torch.equal(eager[1], out[1])


def test_many_requests():
    """More requests than a warp has lanes, with empty ones between."""
    lens = [(37 * i) % 301 for i in range(150)]
    rows = [0 if i % 7 == 3 else 1 + (i % 3 == 0) for i in range(150)]
    lens = [max(n, r) if i % 5 else n for i, (n, r) in enumerate(zip(lens, rows))]
    c = make_cache(lens, 2, 64, 16, torch.int8)
    qs, tokens = starts(rows, extra=3)
    fused = torch.randn(tokens, 12, 64, generator=gen(4), device="cuda").to(torch.float16)
    check_append(c, fused[:, 8:10], fused[:, 10:], qs)
    check_attention(c, fused[:, :8], qs, *call_attention(c, fused[:, :8], qs))


def test_calls_on_two_streams_at_once():
    states = [decode_state(s) for s in (3, 4)]
    want = [decode_step(decode_state(s)) for s in (3, 4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            got[i] = decode_step(states[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_same_inputs_same_bits():
    c = make_cache([5000, 100, 3], 2, 128, 64, torch.float8_e4m3fn)
    qs, tokens = starts([1, 30, 1])
    q = torch.randn(tokens, 8, 128, generator=gen(5), device="cuda").to(torch.bfloat16)
    first = call_attention(c, q, qs)
    s = make_linear(4, 1024, 4096, "pack32", 128, False, False, torch.bfloat16, torch.bfloat16)
    y = call_linear(s)
    for _ in range(5):
        again = call_attention(c, q, qs)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and torch.equal(y, call_linear(s))


def test_nothing_is_written_outside(canary):
    from compressed_tensors_b200 import ops

    with canary():
        for tokens, rows, cols in ((1, 129, 256), (9, 31, 4096), (33, 17, 160)):
            s = make_linear(tokens, rows, cols, "pack32", 32, True, True, torch.bfloat16, torch.bfloat16)
            out = ops.dequantize_linear(s["x"], s["q"], s["scale"], s["zp"], qtype=ops.QINT, col_group=32, scale_row_stride=cols // 32, bias=s["bias"])
            check_linear(s, out)
        for shape in ([(700, 1), (3, 1)], [(300, 130), (64, 1)]):
            c = make_cache([n for n, _ in shape], 2, 128, 16, torch.float8_e4m3fn)
            qs, tokens = starts([m for _, m in shape], extra=1)
            q = torch.randn(tokens, 6, 128, generator=gen(5), device="cuda").to(torch.bfloat16)
            got = ops.kv_cache_attention(q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["seq_lens"], qs, return_lse=True)
            check_attention(c, q, qs, *got)


def test_long_cache_offsets():
    """A page whose first code lies more than 2^32 bytes into the cache."""
    heads, dim, block = 8, 128, 64
    pages = 2 ** 32 // (heads * dim * block) + 40
    c = make_cache([2000], heads, dim, block, torch.int8, spare=0)
    far = {n: torch.zeros(pages, heads, block, dim, dtype=torch.int8, device="cuda") for n in ("k_cache", "v_cache")}
    moved = pages - 1 - c["block_table"][0, :32].long()
    for n in ("k", "v"):
        far[n + "_cache"][moved] = c[n + "_cache"][c["block_table"][0, :32].long()]
        scale = torch.full((pages, heads), 0.02, device="cuda")
        scale[moved] = c[n + "_scale"][c["block_table"][0, :32].long()]
        far[n + "_scale"] = scale
    table = c["block_table"].clone()
    table[0, :32] = moved.to(torch.int32)
    near, there = dict(c), dict(c, block_table=table, **far)
    for rows in (1, 40):
        qs, tokens = starts([rows])
        q = torch.randn(tokens, 32, dim, generator=gen(5), device="cuda").to(torch.bfloat16)
        x, y = call_attention(near, q, qs), call_attention(there, q, qs)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
        check_attention(near, q, qs, *x)


def test_operators_pass_opcheck():
    from compressed_tensors_b200 import torch_ops

    s = make_linear(3, 40, 256, "pack32", 128, True, True, torch.bfloat16, torch.bfloat16)
    c = make_cache([40, 9], 2, 64, 16, torch.int8)
    qs, tokens = starts([1, 3])
    q = torch.randn(tokens, 4, 64, generator=gen(5), device="cuda").to(torch.bfloat16)
    cache = (c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["seq_lens"], qs)
    inputs = {"dequantize_linear": (s["x"], s["q"], s["scale"], s["zp"], 0, 4, 128, 2, "pack32", None, s["bias"]),
              "kv_cache_append": (q[:, :2].contiguous(), q[:, 2:].contiguous(), *cache), "kv_cache_attention": (q, *cache, None, True)}
    assert set(inputs) == set(torch_ops.SERVING_OPERATORS)
    for name, a in inputs.items():
        torch.library.opcheck(getattr(torch.ops.ctb200, name).default, a, test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
