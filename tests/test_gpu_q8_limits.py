"""The 8-bit cache operators at the limits of what they are given: positions behind the rotary tables or the block tables, row starts that
are no row starts, pages that nobody needs any more.  What is skipped is left as it was, what is not is right."""
import pytest
import torch

from q8_plain import IO, Cache, attention_bound, call, quantise, rotate

pytestmark = pytest.mark.gpu


def bits(x):
    return x.cpu().contiguous().view(torch.uint8)


def check_rows(case, got, done):
    """The rows of `done` against the plain form, all others as they were (7)."""
    o, a, spread, floor = case.attend()
    exact_q = case.io != "bf16" and max(case.new) == 1 and case.H // case.N <= 8
    off, bound = (got.double() - o).abs(), attention_bound(case, o, a, spread, floor, exact_q)
    assert bool((off <= bound)[done].all())
    assert bool((got[~done] == 7).all()), "rows that are skipped"


@pytest.mark.parametrize("fmt,io", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("past,new,heads,kv_heads,page,limit", [
    ([40, 60], [1, 1], 4, 2, 16, 50), ([40, 60, 3], [1, 1, 1], 32, 2, 8, 41), ([40, 0, 5], [30, 100, 3], 4, 2, 16, 60),
    ([64, 70], [2, 90], 14, 2, 64, 64), ([3000, 10, 3019], [40, 5, 2], 7, 1, 16, 3020)])
def test_positions_behind_the_rotary_tables_are_skipped(nv, past, new, heads, kv_heads, page, limit, fmt, io):
    """Neither keys nor values are written there, no output either; the rows before them and the other sessions are not touched by it."""
    for what in ("append_attn", "append"):
        case = Cache(past, new, heads, kv_heads, page, fmt, io, layers=1, layer=0, poison=False)
        d = case.device(nv)
        d["cache"].rope_rows = limit
        before = [x.clone() for x in case.codes + case.scales]
        case.append()
        for x, old in zip(case.codes + case.scales, before):
            for s, (p, n) in enumerate(zip(past, new)):
                for t in range(n):
                    if p + t >= limit:
                        ph, slot = case.place(s, p + t)
                        where = (0, ph, slot) if x.dtype == torch.uint8 else (0, ph, slice(None), slot)
                        x[where] = old[where]
        call(nv, d, what)
        torch.cuda.synchronize()
        assert int(d["status"]) == nv.ERR_INVALID
        for x, y in zip(d["codes"] + d["scales"], case.codes + case.scales):
            assert bool((bits(x) == bits(y)).all())
        if what == "append_attn":
            check_rows(case, d["out"].cpu(), case.positions() < limit)


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("far", [200, 2 ** 31 - 17, 2 ** 31 - 9, 0x7ff00000 - 70, 0x7ff00000 - 3, 0x7ff00000, 2 ** 31 - 1, -1, -2 ** 31])
def test_positions_behind_the_block_table(nv, far, window, page):
    """A query whose position has no table entry sees the keys that have one (none: zeros), its own is not written, the status says so; a
    position that is none, or within 2^20 of 2^31, is skipped.  Nothing is walked that is not there: the call takes no longer."""
    for new in ([1, 1, 1], [1, 5, 3]):
        case = Cache([64, 30, 64], new, 6, 2, page, "i8", "bf16", rope="none", layers=1, layer=0, poison=False, seed=page)
        width = 128 // page
        case.tables = case.tables[:, :width].contiguous() if case.tables.shape[1] >= width else torch.nn.functional.pad(
            case.tables, (0, width - case.tables.shape[1]), value=-1)
        d = case.device(nv)
        d["past"][0] = far
        before = [x.clone() for x in case.codes + case.scales]
        case.append()
        ph, slot = case.place(0, 64)
        for x, old in zip(case.codes + case.scales, before):
            where = (0, ph, slot) if x.dtype == torch.uint8 else (0, ph, slice(None), slot)
            x[where] = old[where]
        call(nv, d, "append_attn", window)
        torch.cuda.synchronize()
        skipped = far < 0 or far >= 0x7ff00000
        assert int(d["status"]) == (nv.ERR_INVALID if skipped else nv.ERR_BAD_TABLE)
        for x, y in zip(d["codes"] + d["scales"], case.codes + case.scales):
            assert bool((bits(x) == bits(y)).all())
        got = d["out"].cpu()
        if skipped:
            assert bool((got[0] == 7).all())
        elif window:
            assert bool((got[0] == 0).all())
        else:
            k, v = (case.values(i, 0, 0, page * ((64 + page) // page))[0] for i in (0, 1))
            for h in range(6):       # q, k, weights and v are rounded to fp16, the output to bf16 (attention_bound has the whole account)
                q, kh, vh = case.q[0, h].double(), k[:, h // 3], v[:, h // 3]
                w = torch.softmax((kh @ q) * 128 ** -0.5, -1)
                e = float((kh.abs() @ q.abs()).max()) * 128 ** -0.5 * (2 * 2.0 ** -11 + 2.0 ** -18)
                bound = (w @ vh.abs()) * (2 * (e * (1 + e) + 3 * 2.0 ** -11)) + (w @ vh).abs() * 2.0 ** -8
                assert bool(((got[0, h].double() - w @ vh).abs() <= bound).all())
        case.window = window
        o, a, spread, floor = case.attend()
        off, bound = (got.double() - o).abs(), attention_bound(case, o, a, spread, floor, False)
        assert bool((off <= bound)[1:].all())


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("page", [8, 16, 32, 64])
@pytest.mark.parametrize("window", [1, 7, 24, 100])
def test_pages_behind_the_window_may_be_gone(nv, window, page, fmt):
    """Pages of which no new token sees a key have no entry any more, and what lies in front of the window in the others is NaN: nothing is
    flagged, and nothing of it shows."""
    for past, new in (([200, 207, 31, 64, 111, 8], [1] * 6), ([200, 207, 31, 300, 111], [3, 40, 1, 9, 70])):
        case = Cache(past, new, 4, 2, page, fmt, "bf16", window=window, seed=window)
        gone = []
        for s, p in enumerate(past):
            first = max(0, p - window + 1)
            for j in range(first):
                ph, slot = case.place(s, j)
                for x in case.codes:
                    x[:, ph, slot] = 0x7f
                for x in case.scales:
                    x[:, ph, :, slot] = float("nan")
            gone.append(first // page)
        d = case.device(nv)
        for s, n in enumerate(gone):
            d["tables"][int(case.slices[s]), :n] = -1
        case.append()
        call(nv, d, "append_attn", window)
        torch.cuda.synchronize()
        assert int(d["status"]) == 0
        for i in (0, 1):            # (the plain form multiplies what it does not see by zero)
            x = case.codes[i], case.scales[i]
            bad = x[1].isnan()
            x[0][bad.permute(0, 1, 3, 2)] = 0
            x[1][bad] = 1.0
        check_rows(case, d["out"].cpu(), torch.ones(sum(new), dtype=torch.bool))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("what", ["k inf", "v inf", "k nan", "v nan"])
@pytest.mark.parametrize("window", [0, 200, 40])
def test_cached_rows_that_are_no_numbers_show(nv, fmt, what, window):
    """A cached row with an infinite scale, or with a NaN (e4m3 codes; int8 has none: its scale is NaN here), that all tokens of a chunk see,
    or none (window 40): the outputs of those that see it are no numbers, in the head that has it; all others are right.  Single tokens the
    same."""
    for past, new in (([200, 70, 30], [40, 130, 5]), ([200, 70, 30], [1, 1, 1])):
        case = Cache(past, new, 4, 2, 16, fmt, "bf16", rope="none", window=window, layers=1, layer=0, poison=False)
        i, bad = "kv".index(what[0]), ((0, 150, 1), (1, 0, 0))             # (session, key, kv head)
        d = case.device(nv)
        for s, j, h in bad:
            ph, slot = case.place(s, j)
            if what.endswith("inf"):
                d["scales"][i][0, ph, h, slot] = float("inf")
                d["codes"][i][0, ph, slot, h] = 0
            elif fmt == "e4m3":
                d["codes"][i][0, ph, slot, h, 5] = 0x7f
            else:
                d["scales"][i][0, ph, h, slot] = float("nan")
        case.append()
        call(nv, d, "append_attn", window)
        torch.cuda.synchronize()
        assert int(d["status"]) == 0
        hit = torch.zeros(sum(new), 4, dtype=torch.bool)
        pos, session = case.positions(), torch.repeat_interleave(torch.arange(3), torch.tensor(new))
        for s, j, h in bad:
            hit[:, 2 * h:2 * h + 2] |= ((session == s) & ((pos - window < j) if window else True))[:, None]
        got = d["out"].cpu()
        o, a, spread, floor = case.attend()
        off = (got.double() - o).abs()
        assert bool((off <= attention_bound(case, o, a, spread, floor, False))[~hit].all())
        dim = slice(5, 6) if what == "v nan" and fmt == "e4m3" else slice(None)
        assert bool((~got[hit][:, dim].isfinite()).all())


STARTS = [([1, 1, 1], [0, -50, 10 ** 9, 10 ** 9]), ([1, 1, 1], [7, 3, 2, 1]), ([1, 1, 1], [-3, -2, -1, 0]), ([1, 1, 1], [0, 1, 1, 10 ** 9]),
          ([4, 5, 6], [0, -50, 10 ** 9, 10 ** 9]), ([4, 5, 6], [7, 3, 2, 1]), ([4, 5, 6], [-2 ** 31, 4, 9, 2 ** 31 - 1]), ([4, 5, 6], [15, 15, 15, 15]),
          ([4, 5, 6], [20, 30, 40, 50]), ([4, 5, 6], [2, 3, 3, 8])]


@pytest.mark.parametrize("fmt,io", [("i8", "bf16"), ("e4m3", "f32")])
@pytest.mark.parametrize("new,starts", STARTS)
def test_row_starts_that_are_none_touch_nothing_else(nv, new, starts, fmt, io):
    """tok_start is device data.  Cut to [0, n_tokens], a session has the rows from its start to the next one's, at most max_tokens: those are
    written, read back and attended, and everything else stays: spare rows, guard rows around all buffers, pages of sessions without rows."""
    T, extra = sum(new), 2
    case = Cache([20, 30, 40], new, 4, 2, 16, fmt, io, layers=1, layer=0, poison=False)
    case.qkv = torch.cat((case.qkv, case.qkv[:extra]))
    d = case.device(nv)
    rows = []                                             # (row, session, token) that somebody has
    cut = [min(max(x, 0), T) for x in starts]
    for s in range(3):
        rows += [(r, s, r - cut[s]) for r in range(cut[s], min(max(cut[s + 1], cut[s]), cut[s] + max(new)))]
    d["rows"].n_tokens = T
    d["start"].copy_(torch.tensor(starts, dtype=torch.int32))
    fill = lambda n, *shape, t: torch.full((n + 8, *shape), 7, dtype=t, device="cuda")
    out, back = fill(T, 4, 128, t=d["out"].dtype), [fill(T, 2, 128, t=d["out"].dtype) for _ in range(2)]
    guard = []                                            # pools inside larger buffers
    for name in ("codes", "scales"):
        for i in (0, 1):
            x = d[name][i].flatten()
            big = torch.full((x.numel() + 512,), 7, dtype=x.dtype, device="cuda")
            big[256:-256] = x
            guard.append(big)
            d[name][i] = big[256:-256].view(d[name][i].shape)
    c = d["cache"]
    c.pool_k, c.pool_v, c.scale_k, c.scale_v = (x.data_ptr() for x in d["codes"] + d["scales"])
    ptr = lambda x: x[4:].data_ptr()
    # the plain form: the same rows, session by session, token by token of the order they have
    fresh = [quantise(x, fmt) for x in (rotate(case.qkv[[r for r, _, _ in rows], 4:6], torch.tensor([case.past[s] + t for _, s, t in rows], dtype=torch.long),
                                               case.cs, case.sn, case.rope), case.qkv[[r for r, _, _ in rows], 6:].float())] if rows else []
    for n, (r, s, t) in enumerate(rows):
        ph, slot = case.place(s, case.past[s] + t)
        for i in (0, 1):
            case.codes[i][0, ph, slot] = fresh[i][0][n].view(torch.uint8)
            case.scales[i][0, ph, :, slot] = fresh[i][1][n]
    stream = torch.cuda.current_stream().cuda_stream
    nv.q8_append_attn(c, d["rows"], d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), ptr(out), 0, d["work"].data_ptr(), d["work"].numel(), stream)
    nv.q8_read(c, d["rows"], ptr(back[0]), ptr(back[1]), stream)
    torch.cuda.synchronize()
    assert int(d["status"]) == 0
    for big in guard:
        assert bool((big[:256] == 7).all() and (big[-256:] == 7).all())
    for x, y in zip(d["codes"] + d["scales"], case.codes + case.scales):
        assert bool((bits(x) == bits(y)).all())
    spare = torch.ones(T + 8, dtype=torch.bool)
    spare[[4 + r for r, _, _ in rows]] = False
    for x in [out] + back:
        assert bool((x.cpu()[spare] == 7).all())
    for s in range(3):
        mine = [r for r, o, _ in rows if o == s]
        if not mine:
            continue
        one = Cache([case.past[s]], [len(mine)], 4, 2, 16, fmt, io, layers=1, layer=0, poison=False)
        one.codes, one.scales, one.tables, one.slices, one.cs, one.sn = case.codes, case.scales, case.tables, case.slices[s:s + 1], case.cs, case.sn
        one.q = case.qkv[mine, :4]
        o, a, spread, floor = one.attend()
        off = (out.cpu()[[4 + r for r in mine]].double() - o).abs()
        assert bool((off <= attention_bound(one, o, a, spread, floor, False)).all())
        for i in (0, 1):
            want = one.values(i, 0, one.past[0], one.past[0] + len(mine))[1].to(IO[io])
            assert bool((bits(back[i][[4 + r for r in mine]]) == bits(want)).all())


@pytest.mark.parametrize("new,io", [([1, 1, 1], "f16"), ([30, 0, 9], "bf16")])
def test_pools_of_more_than_four_gigabytes(nv, new, io):
    """The last layer of pools whose offsets pass 32 bits (5 GB of codes each): written, read back, attended."""
    case = Cache([200, 5, 70], new, 16, 8, 16, "i8", io, layers=1, layer=0)
    layer = 5 * 10 ** 9 // case.codes[0].numel()
    d = case.device(nv)
    big = [torch.empty((layer + 1) * x.numel(), dtype=x.dtype, device="cuda") for x in d["codes"] + d["scales"]]
    for b, x in zip(big, d["codes"] + d["scales"]):
        b[-x.numel():] = x.flatten()
    c = d["cache"]
    c.pool_k, c.pool_v, c.scale_k, c.scale_v = (b.data_ptr() for b in big)
    c.layer = layer
    case.append()
    call(nv, d, "append_attn")
    call(nv, d, "read")
    torch.cuda.synchronize()
    assert int(d["status"]) == 0
    for b, x in zip(big, case.codes + case.scales):
        assert bool((bits(b[-x.numel():]) == bits(x.flatten())).all())
    check_rows(case, d["out"].cpu(), torch.ones(sum(new), dtype=torch.bool))
    for got, want in zip(d["back"], case.read()):
        assert bool((bits(got) == bits(want)).all())
    del big
    torch.cuda.empty_cache()
