"""Chunk attention over rows of the 8-bit cache and queries that are small or large as a whole, against plain 64-bit forms (q8_plain.py)."""
import pytest
import torch

from q8_plain import HD, IO, Cache, call

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}        # half a step of the outputs' type, relative
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}     # ... and below its normal range


def run(nv, case, what="append_attn"):
    d = case.device(nv)
    case.append()
    if what == "attn":
        call(nv, d, "append")
    call(nv, d, what, case.window)
    torch.cuda.synchronize()
    assert int(d["status"]) == 0
    for i in (0, 1):
        assert bool((d["codes"][i].cpu() == case.codes[i]).all())
    return d["out"].cpu().double()


def own_value(case):
    """[rows][heads][128]: the value of each query's own key, in 64 bits."""
    v = torch.cat([case.values(1, s, p, p + n)[0] for s, (p, n) in enumerate(zip(case.past, case.new))])
    return v.repeat_interleave(case.H // case.N, dim=1)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("io,top", [("f16", 65504.0), ("bf16", 2.0 ** 17), ("f32", 2.0 ** 17)])
@pytest.mark.parametrize("rope", ["none", "neox", "pairs"])
def test_queries_as_large_as_their_type(nv, io, top, fmt, rope):
    """q up to 2^17 (rotated: fp16's largest numbers by the square root of 2): the scores are finite, and a query that sees its own key alone
    gives its value back: the weight and the value are rounded to fp16 once each (2^-11), the value's scale is in two parts (2^-14)."""
    case = Cache([40, 0, 3], [50, 1, 90], 14, 2, 16, fmt, io, rope=rope, window=1, seed=1)
    sign = torch.where(case.q.float() < 0, -1.0, 1.0)
    case.q.copy_((sign * (top if rope == "none" or io == "f16" else top / 2 ** 0.5 * 0.99)).to(IO[io]))
    case.q[::3] *= 0.6
    got, want = run(nv, case), own_value(case)
    assert bool(got.isfinite().all())
    assert bool(((got - want).abs() <= want.abs() * (2 * 2.0 ** -11 + 2.0 ** -14 + HALF[io]) + 2.0 ** -18).all())
