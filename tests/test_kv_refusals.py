"""What the operators around a key/value cache refuse, through the C ABI and through ``ops``: nothing here needs a GPU, because a refused
call enqueues nothing."""
import ctypes
import math

import pytest
import torch

from arcq_vit_amd import _lib, ops

P = 1 << 20          # an aligned address that nobody follows


def _pages(**kw):
    a = dict(k=P, v=P, k_exponents=None, v_exponents=None, num_pages=4, heads=2, head_dim=64, page_size=16, dtype=_lib.ARCQ_F16)
    a.update(kw)
    return _lib.KvPages(**a)


def _fill(struct, **kw):
    for k, v in kw.items():
        setattr(struct, k, v)
    return struct


def _rotary(**kw):
    a = _lib.QkNormRotaryArgs()
    a.sections[0] = 32
    return _fill(a, **{**dict(dtype=_lib.ARCQ_F16, axes=1, eps=1e-6, magnitude=1.0, tokens=3, q_heads=2, k_heads=1, head_dim=64, pairs=32,
                              q=P, k=P, q_out=P, k_out=P, positions=P, inv_freq=P), **kw})


def _cache(pages=None, **kw):
    return _fill(_lib.KvCacheArgs(), **{**dict(pages=pages or _pages(), k=P, v=P, slots=P, rows=3, k_row_stride=128, k_head_stride=64,
                                               v_row_stride=128, v_head_stride=64, dtype=_lib.ARCQ_F16), **kw})


def _attention(pages=None, **kw):
    return _fill(_lib.AttentionPagedArgs(), **{**dict(pages=pages or _pages(), q=P, out=P, page_table=P, q_offsets=P, kv_lengths=P, workspace=P,
                                                      tokens=3, q_heads=4, sequences=2, table_width=2, table_stride=2, q_token_stride=256,
                                                      q_head_stride=64, out_token_stride=256, out_head_stride=64, scale=0.125,
                                                      dtype=_lib.ARCQ_F16, causal=1), **kw})


@pytest.mark.parametrize("change,code,says", [
    ({"dtype": 3}, -5, b"dtype"), ({"norm": 3}, -6, b"norm"), ({"tokens": -1}, -4, b"negative"), ({"head_dim": 63}, -6, b"head_dim"),
    ({"head_dim": 258}, -6, b"head_dim"), ({"head_dim": 62}, -4, b"pairs"), ({"axes": 0}, -6, b"axes"), ({"axes": 5}, -6, b"axes"),
    ({"pairs": 31}, -4, b"sections"), ({"eps": -1.0}, -4, b"eps"), ({"eps": math.nan}, -4, b"eps"), ({"q": None}, -3, b"NULL"),
    ({"k_out": None}, -3, b"NULL"), ({"positions": None}, -3, b"NULL"), ({"inv_freq": None}, -3, b"NULL"),
    ({"tokens": 1 << 31}, -4, b"too large")])
def test_rotary_refuses(change, code, says):
    lib = _lib.load()
    assert lib.arcq_qk_norm_rotary(ctypes.byref(_rotary(**change)), None) == code
    assert says in lib.arcq_last_error()


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.arcq_qk_norm_rotary(ctypes.byref(_rotary(tokens=0, q=None)), None) == 0
    assert lib.arcq_kv_cache_write(ctypes.byref(_cache(rows=0, k=None)), None) == 0
    assert lib.arcq_kv_cache_read(ctypes.byref(_cache(rows=0, k=None)), None) == 0
    for change in ({"tokens": 0}, {"sequences": 0}):
        assert lib.arcq_attention_paged_fwd(ctypes.byref(_attention(q=None, **change)), None) == 0
        assert lib.arcq_attention_paged_workspace(ctypes.byref(_attention(**change))) == 0
    assert lib.arcq_qk_norm_rotary(None, None) == -3 and lib.arcq_kv_cache_write(None, None) == -3
    assert lib.arcq_attention_paged_fwd(None, None) == -3 and lib.arcq_attention_paged_workspace(None) == -3


_BAD_PAGES = [({"dtype": 0}, -5, b"dtype"), ({"dtype": 2}, -5, b"one dtype"), ({"page_size": 8}, -4, b"page_size"), ({"page_size": 48}, -4, b"page_size"),
              ({"page_size": 0}, -4, b"page_size"), ({"head_dim": 72}, -6, b"head_dim"), ({"head_dim": 272}, -6, b"head_dim"), ({"head_dim": 0}, -6, b"head_dim"),
              ({"num_pages": -1}, -4, b"page_size"), ({"num_pages": 1 << 31}, -4, b"too many"), ({"k": None}, -3, b"NULL"), ({"v": P + 8}, -7, b"aligned"),
              ({"dtype": 3}, -3, b"NULL")]


@pytest.mark.parametrize("change,code,says", _BAD_PAGES)
def test_pages_that_are_refused(change, code, says):
    lib = _lib.load()
    pages = _pages(**change)
    for call in (lambda: lib.arcq_kv_cache_write(ctypes.byref(_cache(pages)), None), lambda: lib.arcq_kv_cache_read(ctypes.byref(_cache(pages)), None),
                 lambda: lib.arcq_attention_paged_fwd(ctypes.byref(_attention(pages)), None)):
        assert call() == code
        assert says in lib.arcq_last_error()


@pytest.mark.parametrize("change,code,says", [
    ({"rows": -1}, -4, b"negative"), ({"dtype": 0}, -5, b"dtype"), ({"k": None}, -3, b"NULL"), ({"slots": None}, -3, b"NULL"), ({"k": P + 2}, -7, b"aligned"),
    ({"v_head_stride": 60}, -7, b"aligned"), ({"k_row_stride": 129}, -7, b"aligned"), ({"rows": 1 << 31}, -4, b"too many")])
def test_cache_refuses(change, code, says):
    lib = _lib.load()
    for fn in (lib.arcq_kv_cache_write, lib.arcq_kv_cache_read):
        assert fn(ctypes.byref(_cache(**change)), None) == code
        assert says in lib.arcq_last_error()


@pytest.mark.parametrize("change,code,says", [
    ({"tokens": -1}, -4, b"negative"), ({"window": -1}, -4, b"negative"), ({"q_heads": 3}, -4, b"divide"), ({"q_heads": 0}, -4, b"divide"),
    ({"window": 5, "causal": 0}, -6, b"window"), ({"scale": 0.0}, -6, b"scale"), ({"scale": -1.0}, -6, b"scale"), ({"scale": math.nan}, -6, b"scale"),
    ({"scale": math.inf}, -6, b"scale"), ({"table_width": 1 << 27}, -4, b"too large"), ({"tokens": 1 << 29}, -4, b"too large"),
    ({"sequences": 1 << 24}, -4, b"too large"), ({"q": None}, -3, b"NULL"), ({"out": None}, -3, b"NULL"), ({"page_table": None}, -3, b"NULL"),
    ({"q_offsets": None}, -3, b"NULL"), ({"kv_lengths": None}, -3, b"NULL"), ({"q": P + 2}, -7, b"aligned"), ({"out_head_stride": 68}, -7, b"aligned"),
    ({"pages": _pages(head_dim=80)}, -6, b"head_dim"), ({"pages": _pages(num_pages=0)}, -4, b"without pages"),
    ({"table_width": 4096, "workspace": None}, -3, b"workspace"), ({"table_width": 4096, "workspace": P + 4}, -3, b"workspace")])
def test_attention_refuses(change, code, says):
    lib = _lib.load()
    assert lib.arcq_attention_paged_fwd(ctypes.byref(_attention(**change)), None) == code
    assert says in lib.arcq_last_error()


def test_grids_of_more_threads_than_an_axis_holds_are_refused():
    lib = _lib.load()
    for fn in (lib.arcq_kv_cache_write, lib.arcq_kv_cache_read):
        assert fn(ctypes.byref(_cache(rows=1 << 29)), None) == -4 and b"too many rows" in lib.arcq_last_error()
    many = _attention(sequences=1 << 23, tokens=1 << 23, table_width=4096)
    assert lib.arcq_attention_paged_fwd(ctypes.byref(many), None) == -4 and b"too many sequences" in lib.arcq_last_error()
    assert lib.arcq_attention_paged_workspace(ctypes.byref(many)) == -4
    # (sizes whose products do not fit 64 bits)
    assert lib.arcq_attention_paged_fwd(ctypes.byref(_attention(tokens=1 << 62)), None) == -4
    assert lib.arcq_attention_paged_fwd(ctypes.byref(_attention(table_width=1 << 60)), None) == -4
    assert lib.arcq_qk_norm_rotary(ctypes.byref(_rotary(tokens=1 << 62, q_heads=2, k_heads=2)), None) == -4


@pytest.mark.parametrize("rows", [(1 << 29) - 31, (1 << 29) - 1])
def test_rows_whose_workgroups_just_fill_an_axis_are_refused(rows):
    """32 rows a workgroup of 256 threads: from 2^29 - 31 rows on there are 2^24 workgroups, 2^32 threads, one more than an axis holds."""
    lib = _lib.load()
    for fn in (lib.arcq_kv_cache_write, lib.arcq_kv_cache_read):
        assert fn(ctypes.byref(_cache(rows=rows)), None) == -4 and b"too many rows" in lib.arcq_last_error()


def test_a_window_of_any_size_is_the_longest_one():
    lib = _lib.load()
    sizes = [lib.arcq_attention_paged_workspace(ctypes.byref(_attention(table_width=4096, window=w))) for w in (0, 1 << 30, (1 << 63) - 1)]
    assert sizes[0] > 0 and sizes == [sizes[0]] * 3


def test_structures_mirror_the_header():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "arcq_hip.h")).read()
    types = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "arcq_kv_pages": _lib.KvPages}
    for name, struct in (("arcq_qk_norm_rotary_args", _lib.QkNormRotaryArgs), ("arcq_kv_pages", _lib.KvPages), ("arcq_kv_cache_args", _lib.KvCacheArgs),
                         ("arcq_attention_paged_args", _lib.AttentionPagedArgs)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1), flags=re.S)
        want = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            m = re.match(r"(?:const )?(int8_t|int32_t|int64_t|float|double|void|arcq_kv_pages) (.*)", decl)
            assert m, decl
            for field in m.group(2).split(","):
                field = field.strip()
                array = re.match(r"(\w+)\[ARCQ_ROTARY_AXES\]", field)
                if array:
                    want.append((array.group(1), types[m.group(1)] * 4))
                else:
                    want.append((field.lstrip("*"), ctypes.c_void_p if field.startswith("*") else types[m.group(1)]))
        assert list(struct._fields_) == want


def test_ops_refuse_host_tensors_and_wrong_shapes():
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    pos, freq = torch.arange(3), torch.ones(32, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rotary(q, k, pos, freq)
    with pytest.raises(RuntimeError, match="norm must be"):
        ops.qk_norm_rotary(q, k, pos, freq, norm="batch")
    with pytest.raises(RuntimeError, match="same tokens"):
        ops.qk_norm_rotary(q, k[:2], pos, freq)
    with pytest.raises(RuntimeError, match="float16, bfloat16 or float32"):
        ops.qk_norm_rotary(q, k.bfloat16(), pos, freq)
    with pytest.raises(RuntimeError, match="float64"):
        ops.qk_norm_rotary(q, k, pos, freq.float())
    with pytest.raises(RuntimeError, match="positions must be int"):
        ops.qk_norm_rotary(q, k, pos.float(), freq)
    with pytest.raises(RuntimeError, match="positions must be \\["):
        ops.qk_norm_rotary(q, k, pos[:2], freq)
    pages = ops.kv_cache_pages(4, 2, 64, 16, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_cache_write(pages, k, k, torch.arange(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_cache_read(pages, torch.arange(3))
    table, off, lens = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attention_paged_fwd(q, pages, table, off, lens)
    for kw in ({"num_pages": -1}, {"heads": 0}, {"head_dim": 24}, {"head_dim": 512}, {"page_size": 8}, {"page_size": 40}, {"dtype": torch.float32}):
        with pytest.raises(RuntimeError):
            ops.kv_cache_pages(**{**dict(num_pages=1, heads=1, head_dim=64, device="cpu"), **kw})


def test_frequencies():
    f, m = ops.rotary_frequencies(32)
    assert f.dtype == torch.float64 and m == 1.0 and f[0] == 1.0 and abs(f[31].item() - 10000.0 ** (-31 / 32)) < 1e-18
    g, _ = ops.rotary_frequencies(32, scaling="linear", factor=4.0)
    assert torch.equal(g * 4.0, f)
    g, _ = ops.rotary_frequencies(32, scaling="base", factor=4.0)
    assert g[0] == 1.0 and abs(g[31].item() * 4.0 / f[31].item() - 1.0) < 1e-12
    g, m = ops.rotary_frequencies(32, scaling="bands", factor=8.0, original=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1] * 8.0, f[turns <= 1], rtol=1e-15)
    assert bool(((g <= f) & (g >= f / 8.0 * (1 - 1e-15))).all()) and abs(m - (1 + 0.1 * math.log(8.0))) < 1e-15
    assert ops.rotary_frequencies(0)[0].shape == (0,)
    for kw in ({"scaling": "other"}, {"scaling": "bands"}, {"base": 0.0}, {"factor": -1.0}):
        with pytest.raises(RuntimeError):
            ops.rotary_frequencies(8, **kw)
