"""What the serving operators refuse, and the index arithmetic of the paged cache on values that a caller may get wrong:
no GPU needed."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "kv_index.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "kv_index_host.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    i64 = ctypes.c_int64
    lib.seq.argtypes = [i64] * 5 + [ctypes.c_void_p]
    lib.written.argtypes = [i64] * 5 + [ctypes.c_int, ctypes.c_void_p]
    lib.most_written.argtypes = [i64] * 3
    lib.most_written.restype = i64
    lib.seen.argtypes = [i64] * 6 + [ctypes.c_int]
    return lib


def test_no_index_leaves_its_buffer(index):
    rng = random.Random(3)
    wild = (-2 ** 31, -7, -1, 0, 1, 5, 63, 64, 65, 1000, 2 ** 31 - 1)
    out = (ctypes.c_int32 * 4)()
    first = ctypes.c_int()
    for _ in range(20000):
        tokens, size = rng.choice((0, 1, 5, 64, 1000)), rng.choice((1, 5, 16, 64))
        capacity = rng.choice((0, 1, 3, 40)) * size
        a = [rng.choice(wild) if rng.random() < 0.7 else rng.randint(0, 80) for _ in range(3)] + [tokens, capacity]
        index.seq(*a, ctypes.addressof(out))
        row, rows, length, start = out
        assert 0 <= row <= tokens and 0 <= rows <= tokens - row
        assert 0 <= length <= capacity and start + rows == max(a[2], 0)
        n = index.written(*a, size, ctypes.addressof(first))
        assert n >= 0
        if n:
            assert 0 <= first.value and (first.value + n) * size <= capacity
            lo = max(start, 0)  # the first and the last written position, and the rows that hold them
            assert row <= row + lo - start <= row + (length - 1) - start < row + rows <= tokens
        for i in (0, rows // 2, rows - 1):
            for causal in (0, 1):
                assert 0 <= index.seen(*a, i, causal) <= length


def test_every_written_block_gets_a_place(index):
    rng = random.Random(4)
    first = ctypes.c_int()
    for _ in range(3000):
        batch, size = rng.randint(1, 20), rng.choice((1, 5, 16, 64))
        rows = [rng.choice((0, 1, 1, 2, rng.randint(0, 300))) for _ in range(batch)]
        tokens = sum(rows) + rng.choice((0, 3))
        at = need = 0
        for n in rows:
            length = n + rng.choice((0, 1, size - 1, rng.randint(0, 500)))
            need += index.written(at, at + n, length, tokens, 1 << 20, size, ctypes.addressof(first))
            at += n
        assert need <= index.most_written(tokens, batch, size)


def _linear(**kw):
    from compressed_tensors_b200 import ops

    a = dict(x=torch.zeros(3, 64, dtype=torch.bfloat16), q=torch.zeros(5, 8, dtype=torch.int32), scale=torch.zeros(5, 2), zp=None, qtype=ops.QINT,
             bits=4, col_group=32, scale_row_stride=2, codec="pack32", global_scale=None, bias=None)
    a.update(kw)
    x, q, scale, zp = a.pop("x"), a.pop("q"), a.pop("scale"), a.pop("zp")
    return ops.dequantize_linear(x, q, scale, zp, **a)


@pytest.mark.parametrize("error, kw", [
    (RuntimeError, {}),  # a CPU tensor
    (NotImplementedError, dict(codec="dtype")),
    (NotImplementedError, dict(bits=8)),
    (NotImplementedError, dict(qtype=1)),
    (TypeError, dict(x=torch.zeros(3, 64))),
    (TypeError, dict(q=torch.zeros(5, 8, dtype=torch.int64))),
    (TypeError, dict(q=torch.zeros(40, dtype=torch.int32))),
    (ValueError, dict(x=torch.zeros((), dtype=torch.bfloat16))),
    (ValueError, dict(x=torch.zeros(3, 72, dtype=torch.bfloat16))),
    (ValueError, dict(col_group=24)),
    (ValueError, dict(col_group=0)),
    (ValueError, dict(scale_row_stride=-1)),
    (ValueError, dict(scale=torch.zeros(5, 1))),
    (TypeError, dict(scale=torch.zeros(5, 2, dtype=torch.float64))),
    (ValueError, dict(zp=torch.zeros(5, 1, dtype=torch.int8))),
    (TypeError, dict(zp=torch.zeros(5, 2, dtype=torch.int32))),
    (NotImplementedError, dict(global_scale=torch.ones(1))),
    (ValueError, dict(bias=torch.zeros(5))),
    (ValueError, dict(bias=torch.zeros(4, dtype=torch.bfloat16))),
    (ValueError, dict(x=torch.zeros(3, 63, dtype=torch.bfloat16), q=torch.zeros(5, 31, dtype=torch.uint8), codec="fp4x2", qtype=1)),
    (NotImplementedError, dict(q=torch.zeros(5, 32, dtype=torch.uint8), codec="fp4x2", qtype=1, zp=torch.zeros(5, 2, dtype=torch.int8))),
    (ValueError, dict(q=torch.zeros(5, 32, dtype=torch.uint8), codec="fp4x2", qtype=1, global_scale=torch.ones(2))),
])
def test_linear_refusals(error, kw):
    with pytest.raises(error):
        _linear(**kw)


def _cache(**kw):
    a = dict(q=torch.zeros(3, 4, 16, dtype=torch.bfloat16), k_cache=torch.zeros(6, 2, 8, 16, dtype=torch.int8),
             v_cache=torch.zeros(6, 2, 8, 16, dtype=torch.int8), k_scale=torch.ones(6, 2), v_scale=torch.ones(6, 2),
             block_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32),
             query_start=torch.zeros(3, dtype=torch.int32))
    a.update(kw)
    return a


BAD_CACHES = [
    (ValueError, dict(k_cache=torch.zeros(6, 2, 8, dtype=torch.int8))),
    (ValueError, dict(v_cache=torch.zeros(6, 2, 4, 16, dtype=torch.int8))),
    (TypeError, dict(k_cache=torch.zeros(6, 2, 8, 16), v_cache=torch.zeros(6, 2, 8, 16))),
    (TypeError, dict(v_cache=torch.zeros(6, 2, 8, 16).to(torch.float8_e4m3fn))),
    (ValueError, dict(k_cache=torch.zeros(6, 2, 16, 8, dtype=torch.int8).transpose(2, 3))),
    (ValueError, dict(k_scale=torch.ones(6, 3))),
    (ValueError, dict(v_scale=torch.ones(6, 2, dtype=torch.float16))),
    (ValueError, dict(k_scale=torch.ones(2, 6).t())),
    (TypeError, dict(seq_lens=torch.zeros(2))),
    (TypeError, dict(block_table=torch.zeros(6, dtype=torch.int32))),
    (ValueError, dict(block_table=torch.zeros(3, 3, dtype=torch.int32))),
    (ValueError, dict(query_start=torch.zeros(2, dtype=torch.int32))),
    (RuntimeError, {}),  # CPU tensors
]


@pytest.mark.parametrize("error, kw", BAD_CACHES + [
    (TypeError, dict(q=torch.zeros(3, 4, 16))),
    (ValueError, dict(q=torch.zeros(3, 3, 16, dtype=torch.bfloat16))),
    (ValueError, dict(q=torch.zeros(3, 4, 8, dtype=torch.bfloat16))),
    (ValueError, dict(q=torch.zeros(12, 16, dtype=torch.bfloat16))),
    (NotImplementedError, dict(q=torch.zeros(3, 4, 320, dtype=torch.bfloat16), k_cache=torch.zeros(6, 2, 8, 320, dtype=torch.int8),
                               v_cache=torch.zeros(6, 2, 8, 320, dtype=torch.int8))),
])
def test_attention_refusals(error, kw):
    from compressed_tensors_b200 import ops

    a = _cache(**kw)
    with pytest.raises(error):
        ops.kv_cache_attention(*a.values())


@pytest.mark.parametrize("error, kw", BAD_CACHES + [
    (TypeError, dict(k=torch.zeros(3, 2, 16), v=torch.zeros(3, 2, 16))),
    (ValueError, dict(v=torch.zeros(3, 2, 16, dtype=torch.float16))),
    (ValueError, dict(v=torch.zeros(4, 2, 16, dtype=torch.bfloat16))),
    (ValueError, dict(k=torch.zeros(3, 4, 16, dtype=torch.bfloat16))),
])
def test_append_refusals(error, kw):
    from compressed_tensors_b200 import ops

    new = torch.zeros(3, 2, 16, dtype=torch.bfloat16)
    a = _cache(**{n: t for n, t in kw.items() if n not in ("k", "v")})
    del a["q"]
    with pytest.raises(error):
        ops.kv_cache_append(kw.get("k", new), kw.get("v", new), *a.values())


def test_c_entry_points_return_a_status():
    """Invalid calls at the C boundary come back with a status; the pointers are never followed."""
    from compressed_tensors_b200 import _lib as L

    lib, one = L.lib(), 16
    good = dict(rows=4, cols=64, col_group=32, row_group=1, scale_row_stride=2, qtype=0, num_bits=4, x_dtype=0, scale_dtype=0, zp_dtype=4, q_dtype=0, codec=1)

    def linear(x=one, tokens=1, q=one, scale=one, zp=None, gs=None, bias=None, out=one, desc=True, **kw):
        d = L.QDesc(**{**good, **kw})
        return lib.ctb_dequantize_linear(ctypes.addressof(d) if desc else None, x, tokens, q, scale, zp, gs, bias, out, None)

    assert linear(desc=False) == 4 and linear(x=None) == 4 and linear(out=None) == 4
    assert linear(tokens=-1) == 1 and linear(col_group=24) == 1 and linear(scale_row_stride=-1) == 1
    assert linear(num_bits=8) == 7 and linear(codec=0) == 7 and linear(row_group=2) == 7 and linear(gs=one) == 7
    assert linear(x_dtype=2) == 2 and linear(scale_dtype=3) == 2 and linear(zp=one, zp_dtype=5) == 2
    assert linear(x=17) == 3
    assert linear(tokens=0) == 0 and linear(rows=0) == 0  # nothing to do, nothing launched

    def cache(**kw):
        f = dict(k=one, v=one, k_scale=one, v_scale=one, num_blocks=4, k_block_stride=256, k_head_stride=256, k_token_stride=16,
                 v_block_stride=256, v_head_stride=256, v_token_stride=16, heads=1, block_size=16, head_dim=16, dtype=4)
        return L.KvCache(**{**f, **kw})

    def batch(**kw):
        f = dict(block_table=one, seq_lens=one, query_start=one, table_width=2, table_stride=2, tokens=1, batch=1)
        return L.KvBatch(**{**f, **kw})

    def attend(c=cache(), b=batch(), q=one, dtype=0, heads=1, out=one, lse=one):
        return lib.ctb_kv_cache_attention(ctypes.addressof(c) if c else None, ctypes.addressof(b), q, dtype, 16, 16, heads, 1.0, 1, out, lse, None, None)

    def append(c=cache(), b=batch(), k=one, v=one, dtype=0):
        return lib.ctb_kv_cache_append(ctypes.addressof(c) if c else None, ctypes.addressof(b), k, v, dtype, 16, 16, 16, 16, None)

    for f in (attend, append):
        assert f(c=None) == 4 and f(c=cache(k=None)) == 4 and f(b=batch(seq_lens=None)) == 4
        assert f(c=cache(dtype=6)) == 2 and f(dtype=2) == 2
        assert f(c=cache(block_size=0)) == 1 and f(c=cache(heads=0)) == 1 and f(b=batch(tokens=-1)) == 1
        assert f(c=cache(head_dim=257)) == 7 and f(b=batch(table_width=1 << 30)) == 7
        assert f(b=batch(tokens=0)) == 0
    assert attend(c=cache(heads=2), heads=3) == 1 and attend(out=None) == 4 and append(k=None) == 4


def test_inputs_that_want_gradients_are_refused():
    from compressed_tensors_b200 import torch_ops as ops

    x = torch.zeros(3, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradients"):
        ops.dequantize_linear(x, torch.zeros(5, 8, dtype=torch.int32), torch.zeros(5, 2), qtype=0, col_group=32, scale_row_stride=2)
    a = _cache()
    a["q"].requires_grad_()
    with pytest.raises(RuntimeError, match="gradients"):
        ops.kv_cache_attention(*a.values())


def test_meta_tensors_give_shapes():
    from compressed_tensors_b200 import torch_ops as ops

    a = {n: t.to("meta") for n, t in _cache().items()}
    out, lse = ops.kv_cache_attention(*a.values(), return_lse=True)
    assert out.is_meta and tuple(out.shape) == (3, 4, 16) and out.dtype == torch.bfloat16 and tuple(lse.shape) == (3, 4) and lse.dtype == torch.float32
    assert ops.kv_cache_append(a["q"][:, :2], a["q"][:, :2], *list(a.values())[1:]) is None
    y = ops.dequantize_linear(torch.empty(2, 3, 64, dtype=torch.float16, device="meta"), torch.empty(5, 8, dtype=torch.int32, device="meta"),
                              torch.empty(5, 2, device="meta"), qtype=0, col_group=32, scale_row_stride=2)
    assert tuple(y.shape) == (2, 3, 5) and y.dtype == torch.float16
