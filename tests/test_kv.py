"""Host-side checks of the paged cache's C ABI (include/ttl_kv.h), without a
GPU: exported symbols, the binding, and the refusals of ttl_kv_create and of
calls without a handle."""
import os
import pathlib
import re

import numpy as np
import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "ttl_kv.h"


def declared_functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(ttl_[a-z0-9_]+)\s*\(", text)))


def test_library_exports_and_binding_cover_header():
    import ttl_moe
    names = declared_functions()
    assert len(names) == 10
    src = (ROOT / "tt-lab_b200" / "python" / "ttl_moe" / "__init__.py").read_text()
    for n in names:
        assert hasattr(ttl_moe.lib(), n), n
        assert f'"{n}"' in src, n


@pytest.mark.parametrize("kw, match", [
    (dict(layers=0), "layers must be"),
    (dict(layers=257), "layers must be"),
    (dict(pages=0), "pages must be"),
    (dict(page_tokens=48), "page_tokens must be"),
    (dict(page_tokens=256), "page_tokens must be"),
    (dict(q_heads=12, kv_heads=8), "multiple of kv_heads"),
    (dict(q_heads=0), "multiple of kv_heads"),
    (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(head_dim=96), "head_dim must be"),
    (dict(rows="bf16", cache="f16"), "cache_type must be"),
    (dict(rows="bf16", cache="f32"), "cache_type must be"),
    (dict(rows="mxfp4"), "rows_type must be"),
    (dict(max_seqs=0), "max_seqs must be"),
    (dict(max_seqs=5000), "max_seqs must be"),
    (dict(max_rows=0), "max_rows must be"),
    (dict(rope_freq=np.ones(4)), "rope_dims must be"),
    (dict(rope_freq=np.ones(64)), "rope_dims must be"),
    (dict(rope_freq=np.array([1.0] * 7 + [np.inf])), "rope_freq must be finite"),
    (dict(rope_freq=np.ones(8), rope_scale=np.nan), "rope_scale must be finite"),
])
def test_create_refuses(kw, match):
    import ttl_moe
    with pytest.raises(RuntimeError, match=match):
        ttl_moe.KvCache(**kw)


def test_unknown_types_are_refused_by_name():
    import ttl_moe
    with pytest.raises(ValueError, match="rows must be one of"):
        ttl_moe.KvCache(rows="f64")
    with pytest.raises(ValueError, match="cache must be one of"):
        ttl_moe.KvCache(cache="int4")


def test_calls_without_a_handle():
    import ttl_moe
    L = ttl_moe.lib()
    assert L.ttl_kv_create(None, None) == ttl_moe.TTL_ERR_ARGUMENT
    assert b"null argument" in L.ttl_kv_last_error(None)
    assert L.ttl_kv_batch_async(None, 1, 1, 1, None, None, None, 1, None, None) == ttl_moe.TTL_ERR_ARGUMENT
    assert L.ttl_kv_append_async(None, 0, 1, None, 0, None, 0, None, 0, None, 0) == ttl_moe.TTL_ERR_ARGUMENT
    assert L.ttl_kv_read_async(None, 0, None, 0, None, 0) == ttl_moe.TTL_ERR_ARGUMENT
    assert L.ttl_kv_attend_async(None, 0, 0, None, 0, None, 0, 0.0, 0.0, None, None) == ttl_moe.TTL_ERR_ARGUMENT
    assert L.ttl_kv_sync(None) == ttl_moe.TTL_ERR_ARGUMENT
    assert L.ttl_kv_page_bytes(None) == 0
    assert L.ttl_kv_stream(None) is None
    L.ttl_kv_destroy(None)


def test_the_default_stream_by_its_handle(monkeypatch):
    """The handle 0, as torch gives it for its default stream, is that stream;
    only None asks for an own one."""
    import types

    import ttl_moe
    seen = []

    def create(cfg, out):
        seen.append(cfg._obj.stream)
        return -1

    monkeypatch.setattr(ttl_moe, "lib", lambda: types.SimpleNamespace(ttl_kv_create=create, ttl_kv_last_error=lambda h: b"no"))
    for stream in (None, 0, 1, 77, types.SimpleNamespace(cuda_stream=0), types.SimpleNamespace(cuda_stream=78)):
        with pytest.raises(RuntimeError, match="no"):
            ttl_moe.KvCache(stream=stream)
    assert seen == [None, 1, 1, 77, 1, 78]


def bare(**kw):
    """A KvCache that has no handle, for its checks of tensors."""
    import torch
    import ttl_moe
    c = ttl_moe.KvCache.__new__(ttl_moe.KvCache)
    c.h, c._i32, c._dtype, c.head_dim, c._rows = None, torch.int32, torch.bfloat16, 64, 1
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_page_tables():
    """A whole table or the leading columns of a wider one; nothing whose rows
    would be read past the memory that holds them."""
    import torch
    c = bare()
    wide = torch.zeros(4, 10, dtype=torch.int32)
    assert c._table_stride(wide, 4) == c._table_stride(wide, 2) == 10
    assert c._table_stride(wide[:, :3], 4) == c._table_stride(wide[:3, :1], 3) == 10
    assert c._table_stride(wide[2:, :7], 2) == 10
    assert c._table_stride(wide[1:2, 4:6], 1) == 2      # one row is read as far as it goes
    assert c._table_stride(wide[:3, 4:6], 3) == 10      # another row follows the last
    assert c._table_stride(torch.zeros(4, 1, dtype=torch.int32), 4) == 1
    for bad in (wide[:, 4:6], wide[1:, 1:3], wide[:, ::2], wide.T, wide.long(), wide[0], wide[:3],
                wide[:1, :2].expand(4, 2), torch.zeros(40, dtype=torch.int32).as_strided((4, 10), (5, 1))):
        with pytest.raises(ValueError, match="pages must be"):
            c._table_stride(bad, 4)


def test_one_row_has_no_stride():
    """A single row of rows that are no multiple of 16 bytes apart, an expanded
    one, and one whose stride torch made up."""
    import torch
    c = bare()
    x = torch.zeros(3, 700, dtype=torch.bfloat16)
    for t in (x.as_strided((1, 8, 64), (700, 64, 1)), x[:1, :512].unflatten(1, (8, 64)), torch.zeros(1, 1, 8, 64, dtype=torch.bfloat16).expand(1, 1, 8, 64)[0],
              torch.zeros(8, 64, dtype=torch.bfloat16).as_strided((1, 8, 64), (1, 64, 1))):
        assert c._row_array(t, "q", 8) == (t.data_ptr(), 512)
    assert c._row_array(x[:, :512].unflatten(1, (8, 64)), "q", 8) == (x.data_ptr(), 700)


@pytest.mark.skipif(os.path.exists("/dev/nvidia0"), reason="a GPU is present")
def test_create_without_gpu_fails_loudly():
    import ttl_moe
    with pytest.raises(RuntimeError, match="no CUDA device"):
        ttl_moe.KvCache()


def test_gptoss_rope_is_the_models_table():
    """gptoss_rope against the float table of the oracle's restatement of the
    GptOssModel constructor: equal to a few f32 steps (powf, logf)."""
    import oracle
    import ttl_moe
    freq, scale = ttl_moe.gptoss_rope()
    assert np.allclose(freq, oracle.rope_frequencies(), rtol=16 * 2.0 ** -24, atol=0)
    assert abs(scale - (1 + 0.1 * np.log(32.0))) < 1e-12


def test_plain_mxfp4_rounds_to_nearest_even():
    """The tests' own 4-bit form: borders between codes, saturation, zeros."""
    import torch

    from kv_plain import mxfp4
    x = torch.zeros(32, dtype=torch.float64)
    x[0] = 4.0  # scale 1
    x[1:12] = torch.tensor([0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.9, -2.5])
    want = [4, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, -2]
    assert mxfp4(x)[:12].tolist() == want
    assert (mxfp4(torch.zeros(32)) == 0).all()
    x[20] = float("inf")
    assert torch.isnan(mxfp4(x)).all()
