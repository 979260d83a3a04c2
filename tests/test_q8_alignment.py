"""Tables, positions and row starts of the 8-bit cache operators that are not on a 4-byte boundary are refused on the host (no GPU needed)."""
import pytest

from test_q8_refusals import parts


@pytest.mark.parametrize("where,field", [("cache", "tables"), ("cache", "slice_ids"), ("cache", "status"), ("rows", "n_past"), ("rows", "tok_start")])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_integers(nv, where, field, off):
    cache, rows, p, keep = parts(nv)
    setattr(cache if where == "cache" else rows, field, p + off)
    L, before = nv.lib, nv.lib.nova_launch_count()
    assert L.nova_launch_q8_append(cache, rows, p, p, None) == nv.ERR_INVALID
    assert L.nova_launch_q8_read(cache, rows, p, p, None) == nv.ERR_INVALID
    assert L.nova_launch_q8_attn(cache, rows, p, p, 0, p, 1 << 40, None) == nv.ERR_INVALID
    assert L.nova_launch_q8_append_attn(cache, rows, p, p, p, p, 0, p, 1 << 40, None) == nv.ERR_INVALID
    assert L.nova_launch_count() == before
