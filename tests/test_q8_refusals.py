"""Calls of the 8-bit cache operators that are refused on the host, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest


def parts(nv, **over):
    shape = nv.KvShape(28, 4, 128, 16, nv.KV_I8, 1)
    buf = C.create_string_buffer(4096 + 16)
    p = (C.addressof(buf) + 15) & ~15                        # host memory: these calls never get as far as a launch
    cache = nv.Q8Cache(shape=shape, layer=0, nb=8, pool_k=p, pool_v=p, scale_k=p, scale_v=p, tables=p, table_stride=4, slice_ids=None,
                       rope_cs=p, rope_sn=p, rope_rows=64, status=None)
    rows = nv.Q8Rows(n_sessions=2, n_tokens=2, max_tokens=1, io_dtype=nv.IO_F16, n_past=p, tok_start=None)
    return cache, rows, p, buf


CACHE = [("layer", -1, "INVALID"), ("nb", 0, "INVALID"), ("pool_k", None, "INVALID"), ("pool_v", 8, "INVALID"), ("scale_k", None, "INVALID"),
         ("scale_v", 4, "INVALID"), ("tables", None, "INVALID"), ("table_stride", 0, "INVALID"), ("rope_cs", None, "INVALID"),
         ("rope_rows", 0, "INVALID"), ("nb", 2 ** 30, "TOO_LARGE"), ("layer", 2 ** 28, "TOO_LARGE")]
SHAPE = [("kv_dtype", 0, "UNSUPPORTED"), ("kv_dtype", 1, "UNSUPPORTED"), ("kv_dtype", 9, "UNSUPPORTED"), ("head_dim", 64, "UNSUPPORTED"),
         ("kv_block", 24, "UNSUPPORTED"), ("n_heads", 27, "INVALID"), ("n_kv_heads", 0, "INVALID"), ("n_heads", 4 * 129, "UNSUPPORTED")]
ROWS = [("n_sessions", -1, "INVALID"), ("n_tokens", -1, "INVALID"), ("n_tokens", 3, "INVALID"), ("max_tokens", 2, "INVALID"), ("io_dtype", 3, "UNSUPPORTED"),
        ("n_past", None, "INVALID"), ("q_stride", 28 * 128 - 8, "INVALID"), ("k_stride", 4 * 128 + 4, "INVALID"), ("v_stride", 128, "INVALID"),
        ("out_stride", -3584, "INVALID")]


@pytest.mark.parametrize("where,field,value,code", [("cache",) + x for x in CACHE] + [("shape",) + x for x in SHAPE] + [("rows",) + x for x in ROWS])
def test_bad_descriptors(nv, where, field, value, code):
    cache, rows, p, keep = parts(nv)
    setattr({"cache": cache, "shape": cache.shape, "rows": rows}[where], field, value)
    want = getattr(nv, "ERR_" + code)
    L = nv.lib
    assert L.nova_launch_q8_append(cache, rows, p, p, None) == want
    assert L.nova_launch_q8_read(cache, rows, p, p, None) == want
    assert L.nova_launch_q8_attn(cache, rows, p, p, 0, p, 1 << 40, None) == want
    assert L.nova_launch_q8_append_attn(cache, rows, p, p, p, p, 0, p, 1 << 40, None) == want


def test_values_of_codes(nv):
    import numpy as np
    import torch
    c = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    assert np.array_equal(nv.q8_values(c.numpy(), nv.KV_E4M3), c.view(torch.float8_e4m3fn).float().numpy(), equal_nan=True)
    assert np.array_equal(nv.q8_values(c.numpy(), nv.KV_I8), c.view(torch.int8).float().numpy())


def test_bad_pointers_and_sizes(nv):
    cache, rows, p, keep = parts(nv)
    L, bad = nv.lib, nv.ERR_INVALID
    for k, v in ((None, p), (p, None), (p + 2, p), (p, p + 8)):
        assert L.nova_launch_q8_append(cache, rows, k, v, None) == bad
        assert L.nova_launch_q8_read(cache, rows, k, v, None) == bad
    need = nv.q8_workspace_bytes(cache.shape, rows)
    for q, out, window, work, size in ((None, p, 0, p, 1 << 40), (p, None, 0, p, 1 << 40), (p + 2, p, 0, p, 1 << 40), (p, p + 4, 0, p, 1 << 40),
                                       (p, p, -1, p, 1 << 40), (p, p, 0, p + 8, 1 << 40)) + (((p, p, 0, None, 1 << 40), (p, p, 0, p, need - 1)) if need else ()):
        assert L.nova_launch_q8_attn(cache, rows, q, out, window, work, size, None) == bad
        assert L.nova_launch_q8_append_attn(cache, rows, q, p, p, out, window, work, size, None) == bad
    assert L.nova_launch_q8_append_attn(cache, rows, p, None, p, p, 0, p, 1 << 40, None) == bad
    assert L.nova_launch_q8_append(None, rows, p, p, None) == bad and L.nova_launch_q8_append(cache, None, p, p, None) == bad
    assert L.nova_q8_workspace_bytes(None, rows) == 0 and L.nova_q8_workspace_bytes(cache.shape, None) == 0
    rows.tok_start, rows.max_tokens = p, 0
    assert L.nova_launch_q8_append(cache, rows, p, p, None) == bad


def test_nothing_to_do(nv):
    """No sessions, or no rows: nothing is launched, and no buffer is asked for."""
    cache, rows, p, keep = parts(nv)
    rows.n_tokens = rows.max_tokens = 0
    for n in (0, 2):
        rows.n_sessions = n
        before = nv.lib.nova_launch_count()
        assert nv.lib.nova_launch_q8_append(cache, rows, None, None, None) == 0
        assert nv.lib.nova_launch_q8_read(cache, rows, None, None, None) == 0
        assert nv.lib.nova_launch_q8_attn(cache, rows, None, None, 0, None, 0, None) == 0
        assert nv.lib.nova_launch_q8_append_attn(cache, rows, None, None, None, None, 0, None, 0, None) == 0
        assert nv.lib.nova_launch_count() == before
