"""Chunk attention over rows of the 8-bit cache and queries that are small or large as a whole, against plain 64-bit forms (q8_plain.py)."""
import pytest
import torch

from q8_plain import HD, IO, Cache, attention_bound, call

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


# What fp16 operands leave of a value: it is rounded once (2^-11), and its scale is in two parts (2^-22, as is the rounding of the product
# with the second one).  fp16's grid ends at 2^-24: the scale, 64 (256) times as large, is off by 2^-25, which the code, 127 / 64 (448 / 256) at
# the most, makes 2^-24; the product and the product with the second part are off by 2^-25 each.  A key goes in over 2.
VALUE, VALUE_LOW = 2.0 ** -11 + 2.0 ** -20, 2.0 ** -23
KEY, KEY_LOW = VALUE, 2.0 ** -22
SMALL = [1.0, 0.1, 1e-2, 1e-3, 1e-4, 1e-5]


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("io,size", [(io, m) for m in SMALL for io in ("bf16", "f32", "f16") if io != "f16" or m > 1e-4])
def test_values_of_any_size(nv, io, size, fmt):
    """A query that sees its own key alone gives its value back, with the weight rounded to fp16 once (2^-11)."""
    for new, heads, kv_heads, page in (([70, 3, 1, 130], 14, 2, 16), ([5, 9], 6, 3, 8), ([1, 1], 16, 1, 64)):
        case = Cache([40, 0, 7, 20][:len(new)], new, heads, kv_heads, page, fmt, io, window=1, seed=len(new))
        case.v.copy_((case.v.float() * size).to(IO[io]))
        case.scales[1] *= size
        got, want = run(nv, case), own_value(case)
        off, bound = (got - want).abs(), want.abs() * (2.0 ** -11 + VALUE + HALF[io]) + VALUE_LOW + TINY[io]
        assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_sizes_that_change_along_the_keys(nv, fmt):
    """Values of one size after those of another, in runs that begin and end inside a tile: each query sees the last 8 keys, which weigh
    the same (q is zero: the weights are powers of two)."""
    n = 400
    sizes = torch.tensor([1.0, 1e-3, 1e-6, 30.0, 1e-2])[torch.arange(n) // 37 % 5]
    case = Cache([0, 13], [n, 60], 4, 2, 16, fmt, "f32", window=8, seed=4)
    case.q.zero_()
    case.v[:n] *= sizes[:, None, None]
    got = run(nv, case)
    at = 0
    for s, (p, m) in enumerate(zip(case.past, case.new)):
        v = case.values(1, s, 0, p + m)[0]
        for t in range(m):
            w = v[max(0, p + t - 7):p + t + 1]
            bound = w.abs().mean(0) * (VALUE + 2.0 ** -20) + VALUE_LOW + w.mean(0).abs() * HALF["f32"]
            off = (got[at + t].view(2, 2, HD) - w.mean(0)[:, None]).abs()
            assert bool((off <= bound[:, None]).all()), (s, t, float((off / bound[:, None]).max()))
        at += m


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("io,size", [(io, m) for m in SMALL[:5] for io in ("bf16", "f32", "f16") if io != "f16" or m > 1e-4])
def test_keys_of_any_size(nv, io, size, fmt):
    """Small keys and queries as much larger, all of one sign, so that a row's error moves its score as a whole."""
    case = Cache([30, 0, 9], [40, 2, 100], 6, 2, 16, fmt, io, rope="none", seed=2, poison=False)
    case.k.copy_((case.k.float().abs() * size).to(IO[io]))
    case.q.copy_((case.q.float().abs() * (0.7 / size)).to(IO[io]))
    c = case.typed(case.codes[0]).float().abs()
    case.codes[0] = (c.to(torch.int8) if fmt == "i8" else c.to(torch.float8_e4m3fn)).view(torch.uint8)
    case.scales[0] *= size
    got = run(nv, case)
    o, a, spread, floor = case.attend()
    q = case.q.double().abs().sum(-1) * HD ** -0.5
    # a score: q rounded to fp16 (2^-11), the key, 17 additions of the product's sum; then as anywhere: a score off by e moves the quotient
    # by 2 e (1 + e) of the sum of |v|, weights and values are rounded once each
    e = spread * (2.0 ** -11 + KEY + 2.0 ** -19 + 2.0 ** -22) + q * KEY_LOW
    bound = a * (2 * (e * (1 + e) + 2.0 ** -11 + VALUE) + 2.0 ** -16)[..., None] + VALUE_LOW + floor * 2.0 ** -32 + o.abs() * HALF[io] + TINY[io]
    off = (got - o).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5])
def test_prefill_of_an_engine(nv, fmt, size):
    """nova_batch_prefill on 8-bit pools: the bound of test_values_of_any_size, fp32 activations."""
    H, N, n = 6, 2, 90
    kvd = nv.KV_I8 if fmt == "i8" else nv.KV_E4M3
    eng = nv.Engine(1, H, N, ctx=128, n_slices=2, kv_dtype=kvd)
    b = eng.batch([eng.session_create(), eng.session_create()])
    b.set_window(1)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, n, h, HD, generator=g) for h in (H, N, N))
    v *= size
    dev = [nv.to_device(x.numpy()) for x in (q, k, v)]
    out = nv.DevBuf(q.numel() * 4)
    b.prefill(0, n, *(x.ptr for x in dev), out.ptr)
    nv.check(nv.lib.dev_sync())
    assert b.device_status() == 0
    got = torch.from_numpy(out.download("float32").reshape(2, n, H, HD)).double()
    codes, scales = eng.read_pools()[1], eng.read_scales()[1]
    wide = nv.q8_values(codes, kvd)[0].astype("float64") * scales[0].swapaxes(1, 2)[..., None]              # [pages][page][kv heads][128]
    for s in (0, 1):
        table = eng.pool.table(eng.session_slice(b.sessions[s]))
        want = torch.from_numpy(wide)[[int(table[j // 16]) for j in range(n)], [j % 16 for j in range(n)]].repeat_interleave(H // N, dim=1)
        assert bool(((got[s] - want).abs() <= want.abs() * (2.0 ** -11 + VALUE + HALF["f32"]) + VALUE_LOW).all())
    b.close()
    eng.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("mean", [0.0, 2.0, 6.0])
def test_single_tokens_over_keys_with_one_large_number(nv, mean, io, fmt):
    """Keys whose codes are small but for one (the scale is that one's), queries of mostly one sign: q is taken in two fp16 parts, so a score
    is off by 2^-18 of sum |q k| at the most, whatever sum q is."""
    past = [3, 7, 15, 2, 40, 5, 1, 6] * 4
    case = Cache(past, [1] * len(past), 14, 2, 16, fmt, io, rope="none", seed=int(mean), poison=False, layers=1, layer=0)
    g = torch.Generator().manual_seed(9)
    case.q.copy_((torch.randn(case.q.shape, generator=g) * 0.5 + mean).to(IO[io]))
    shape = case.codes[0].shape
    small = torch.randint(-3, 4, shape, generator=g).float()
    small[..., 77] = 127.0 if fmt == "i8" else 448.0
    case.codes[0] = (small.to(torch.int8) if fmt == "i8" else small.to(torch.float8_e4m3fn)).view(torch.uint8)
    case.scales[0].fill_(0.04)
    case.k.copy_((torch.randint(-3, 4, case.k.shape, generator=g).float() * 0.04).to(IO[io]))
    case.k[..., 77] = (127.0 if fmt == "i8" else 448.0) * 0.04
    got = run(nv, case)
    o, a, spread, floor = case.attend()
    bound = attention_bound(case, o, a, spread, floor, True)
    assert bool(((got - o).abs() <= bound).all()), f"{float(((got - o).abs() / bound).max()):.3g} of the bound"
