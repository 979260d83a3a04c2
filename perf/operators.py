"""Measured cases of the 8-bit paged KV cache: writing it, reading it back, decode and chunk attention over it.

The cache holds one code of 8 bits per value (int8, or e4m3) and one fp32 scale per token and kv head:
    value = code * scale,  scale = max(|row|, 2^-60) / Q,  code = round(row * (Q / max(|row|, 2^-60))),  Q = 127 or 448
(which code a value next to a border gets is decided in fp32: the quotient, then the product, each rounded once)
in pages of `page` tokens behind a block table: codes [pages][page][kv heads][128], scales [pages][kv heads][page].

A case names its operator:
  store   append new tokens of every session (keys rotated, both quantised), then read the same rows back
  read    read a range of every session's rows back
  decode  append ONE new token per session and attend with it over all the session's keys
  chunk   append a chunk of new tokens per session (their number differs) and attend causally, or in a sliding window
"""
import math

import torch

own = False

HD = 128
Q_MAX = {"i8": 127.0, "e4m3": 448.0}
IO = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
MIN_AMAX = 2.0 ** -60


# ------------------------------------------------------------------------------------------------- cases
def _case(op, sessions, ctx, new, heads, kv_heads, page, fmt, io, window=0, packed=False, rope="neox"):
    return {"op": op, "sessions": sessions, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "heads": heads,
            "kv_heads": kv_heads, "page": page, "fmt": fmt, "io": io, "window": window, "packed": packed, "rope": rope}


def listed():
    cases = {
        # one user's short conversation: a step is all latency
        "decode 1x1024 12h2": _case("decode", 1, (1024, 1024), (1, 1), 12, 2, 16, "i8", "f16"),
        # a few conversations of different lengths, q/k/v as one projection's output
        "decode 8x2k-8k 28h4": _case("decode", 8, (2048, 8192), (1, 1), 28, 4, 16, "e4m3", "bf16", packed=True),
        # a full server: many long conversations
        "decode 64x8192 40h8": _case("decode", 64, (8192, 8192), (1, 1), 40, 8, 16, "i8", "bf16"),
        # one very long document, the framework's own fp32 activations
        "decode 1x131072 28h4": _case("decode", 1, (131072, 131072), (1, 1), 28, 4, 32, "i8", "f32"),
        # drafted tokens of a speculative step, between none and eight per session
        "chunk 16x(0-8) over 2k-8k": _case("chunk", 16, (2048, 8192), (0, 8), 28, 4, 16, "i8", "bf16"),
        # prompts arriving in chunks beside one another, ragged
        "chunk 8x(301-512) over 2k-8k": _case("chunk", 8, (2048, 8192), (301, 512), 28, 4, 16, "e4m3", "f16", packed=True),
        # a long prompt's next chunk
        "chunk 1x2048 over 16384": _case("chunk", 1, (16384, 16384), (2048, 2048), 40, 8, 64, "i8", "bf16"),
        # fresh prompts, sliding window, pairs rotated next to one another
        "chunk 5x(1-1021) window 512": _case("chunk", 5, (0, 1500), (1, 1021), 12, 2, 32, "e4m3", "bf16", window=512, rope="pairs"),
        # one step's tokens of a small batch
        "store 8x1": _case("store", 8, (2048, 8192), (1, 1), 28, 4, 16, "i8", "f16"),
        # whole prompts moved into the cache
        "store 16x(1000-4096)": _case("store", 16, (0, 300), (1000, 4096), 40, 8, 16, "e4m3", "bf16", packed=True),
        # a short conversation handed to another engine
        "read 1x1000": _case("read", 1, (24, 24), (1000, 1000), 12, 2, 64, "e4m3", "f32"),
        # many conversations handed over at once
        "read 32x(513-4608)": _case("read", 32, (0, 0), (513, 4608), 28, 4, 16, "i8", "bf16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "chunk", "chunk", "store", "read"])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8])
    io = rng.choice(["f16", "bf16", "f32"])
    common = (group * kv_heads, kv_heads, rng.choice([8, 16, 32, 64]), rng.choice(["i8", "e4m3"]))
    packed, rope = rng.random() < 0.5, rng.choice(["neox", "neox", "pairs", "none"])
    if op == "decode":
        sessions = _log(rng, 1, 64)
        hi = _log(rng, 1, min(131072, 4_000_000 // (sessions * kv_heads)))
        return _case(op, sessions, (rng.randint(0, hi), hi), (1, 1), *common, io, rng.choice([0, 0, 0, 777]), packed, rope)
    if op == "chunk":
        # chunks go through fp16 weights: activations of 16 bits
        sessions, new = _log(rng, 1, 16), _log(rng, 2, 1024)
        most = 150_000_000 // (sessions * new * group * kv_heads)
        hi = min(_log(rng, 16, 16384), max(16, most))
        return _case(op, sessions, (rng.randint(0, hi), hi), (rng.randint(0, new), new), *common, rng.choice(["f16", "bf16"]),
                     rng.choice([0, 0, 0, 300]), packed, rope)
    sessions = _log(rng, 1, 32)
    new = _log(rng, 1, max(2, min(8192, 400_000 // (sessions * kv_heads))))
    return _case(op, sessions, (rng.randint(0, 300), 300), (rng.randint(0, new), new), *common, io, 0, packed, rope)


def _spread(lo, hi, n, salt):
    """n whole numbers between lo and hi, the same for every seed."""
    return [lo + int(((i + 1) * 0.6180339887498949 + salt) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _lens(case):
    past = _spread(case["ctx_lo"], case["ctx_hi"], case["sessions"], 0.11)
    new = _spread(case["new_lo"], case["new_hi"], case["sessions"], 0.37)
    if not sum(new):
        new[0] = max(1, case["new_hi"])
    return past, new


def work(case):
    past, new = _lens(case)
    H, N, io = case["heads"], case["kv_heads"], IO[case["io"]].itemsize
    rows = sum(new)
    row_q8, row_io = 2 * N * (HD + 4), 2 * N * HD * io
    if case["op"] == "store":
        return {"bytes": rows * 2 * (row_q8 + row_io), "flops": rows * N * HD * 12}
    if case["op"] == "read":
        return {"bytes": rows * (row_q8 + row_io), "flops": rows * N * HD * 2}
    w = case["window"]
    keys = seen = 0
    for p, n in zip(past, new):
        if not n:
            continue
        first = max(0, p - w + 1) if w else 0
        keys += p - first                                   # cached keys that some new token sees
        seen += sum(min(w, p + t + 1) if w else p + t + 1 for t in range(n))
    return {"bytes": keys * row_q8 + rows * (row_io + row_q8 + 2 * H * HD * io), "flops": 4 * HD * H * seen}


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    past, new = _lens(case)
    S, H, N, page, fmt, io = case["sessions"], case["heads"], case["kv_heads"], case["page"], case["fmt"], IO[case["io"]]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    need = [(p + n + page - 1) // page for p, n in zip(past, new)]
    pages, width = sum(need) + 3, max(need) + 1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    # sessions keep their tables in any order of slices
    slices = torch.randperm(S, generator=g, device=dev).to(torch.int32)
    tables = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, c in enumerate(need):
        tables[slices[s].long(), :c] = order[at:at + c]
        at += c

    def pool():
        x = torch.randn(pages, page, N, HD, generator=g, device=dev, dtype=torch.float16)
        if fmt == "i8":
            codes = x.mul_(47).round_().clamp_(-127, 127).to(torch.int8)
        else:
            codes = x.mul_(166).clamp_(-448, 448).to(torch.float8_e4m3fn)
        spread = torch.randn(pages, N, page, generator=g, device=dev)
        return codes, torch.exp(spread * 0.4) / (47 if fmt == "i8" else 166)

    k_codes, k_scales = pool()
    v_codes, v_scales = pool()
    T = sum(new)
    qkv = torch.randn(T, H + 2 * N, HD, generator=g, device=dev).mul_(1.3).to(io)
    q, k, v = qkv[:, :H], qkv[:, H:H + N], qkv[:, H + N:]
    if not case["packed"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    rows = max(p + n for p, n in zip(past, new)) + 1
    angle = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * torch.exp(
        torch.arange(HD // 2, dtype=torch.float64, device=dev) * (-math.log(1e6) / (HD // 2)))
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return {
        "case": dict(case), "codes": (k_codes, v_codes), "scales": (k_scales, v_scales), "tables": tables, "slices": slices,
        "past": torch.tensor(past, dtype=torch.int32, device=dev), "start": torch.tensor(start, dtype=torch.int32, device=dev),
        "q": q, "k": k, "v": v, "cos": angle.cos().float(), "sin": angle.sin().float(), "rows": T, "longest": max(new),
        "most_keys": max(p + n for p, n in zip(past, new)), "uniform": min(new) == max(new),
        "out": torch.empty(T, H, HD, dtype=io, device=dev) if case["op"] in ("decode", "chunk") else None,
        "back": (torch.empty(T, N, HD, dtype=io, device=dev), torch.empty(T, N, HD, dtype=io, device=dev)) if case["op"] in ("store", "read") else None,
    }


# ------------------------------------------------------------------------------------------------- plain forms
def _places(state):
    """Of every new row: its session, its position, its page and its slot within the page."""
    start, page = state["start"].long(), state["case"]["page"]
    row = torch.arange(state["rows"], device=start.device)
    s = torch.searchsorted(start, row, right=True) - 1
    pos = state["past"].long()[s] + row - start[s]
    phys = state["tables"][state["slices"].long()[s], pos // page].long()
    return s, pos, phys, pos % page


def _rotate(x, pos, state):
    """Pairs turned by their position's angle; product and sum are rounded once (fused), as a multiply-add does."""
    if state["case"]["rope"] == "none":
        return x.float()
    x = x.float()
    c, s = state["cos"][pos][:, None], state["sin"][pos][:, None]
    a, b = (x[..., :64], x[..., 64:]) if state["case"]["rope"] == "neox" else (x[..., 0::2], x[..., 1::2])
    u = (a.double() * c.double() - (b * s).double()).float()
    w = (a.double() * s.double() + (b * c).double()).float()
    return torch.cat((u, w), -1) if state["case"]["rope"] == "neox" else torch.stack((u, w), -1).flatten(-2)


def _write(state, which, rows, phys, slot):
    fmt = state["case"]["fmt"]
    amax = rows.abs().amax(-1).clamp_min(MIN_AMAX)
    top = torch.full_like(amax, Q_MAX[fmt])              # (a tensor over a tensor: one rounded division, with no reciprocal between)
    scaled = rows * (top / amax)[..., None]
    codes = scaled.round().to(torch.int8) if fmt == "i8" else scaled.to(torch.float8_e4m3fn)
    state["codes"][which].view(torch.uint8)[phys, slot] = codes.view(torch.uint8)
    state["scales"][which][phys, :, slot] = amax / top


def _append(state):
    _, pos, phys, slot = _places(state)
    _write(state, 0, _rotate(state["k"], pos, state), phys, slot)
    _write(state, 1, state["v"].float(), phys, slot)


def _values(state, which, phys, slot):
    codes = state["codes"][which]
    return codes.view(torch.uint8)[phys, slot].view(codes.dtype).float() * state["scales"][which][phys, :, slot][..., None]


def _read(state):
    _, _, phys, slot = _places(state)
    io = IO[state["case"]["io"]]
    return _values(state, 0, phys, slot).to(io), _values(state, 1, phys, slot).to(io)


def _attend(state):
    case, dev = state["case"], state["q"].device
    S, H, N, page, T = case["sessions"], case["heads"], case["kv_heads"], case["page"], state["longest"]
    G, M = H // N, state["most_keys"]
    start, past = state["start"].long(), state["past"].long()
    key = torch.arange(M, device=dev)
    held = key[None] < (past + start[1:] - start[:-1])[:, None]                                    # [S, M]
    phys = state["tables"][state["slices"].long()][:, key // page].long().clamp_min(0)
    k, v = (_values(state, i, phys, (key % page).expand(S, M)) for i in (0, 1))                    # [S, M, N, HD]
    k, v = (x.masked_fill(~held[..., None, None], 0.0).permute(0, 2, 1, 3) for x in (k, v))        # [S, N, M, HD]
    tok = torch.arange(T, device=dev)
    real = tok[None] < (start[1:] - start[:-1])[:, None]                                           # [S, T]
    row = (start[:-1, None] + tok[None]).clamp_max(state["rows"] - 1)
    pos = past[:, None] + tok[None]
    q = _rotate(state["q"][row.flatten()], pos.flatten().clamp_max(state["cos"].shape[0] - 1), state)
    q = q.view(S, T, N, G, HD).permute(0, 2, 3, 1, 4).reshape(S, N, G * T, HD)
    seen = (key <= pos[..., None]) & held[:, None]                                                 # [S, T, M]
    if case["window"]:
        seen = seen & (key > pos[..., None] - case["window"])
    score = (q @ k.transpose(-1, -2)).view(S, N, G, T, M).mul_(1 / math.sqrt(HD)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    o = (weight.view(S, N, G * T, M) @ v).view(S, N, G, T, HD) / total.clamp_min(1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, T, H, HD)
    return o[real].to(IO[case["io"]])


# ------------------------------------------------------------------------------------------------- the framework's operators
def _package():
    from __graft_entry__ import load_package
    return load_package()


def _handle(state):
    """What a program keeps beside its cache: the descriptors of cache and rows, and the attention's workspace."""
    if "handle" not in state:
        nv, case = _package(), state["case"]
        shape = nv.KvShape(case["heads"], case["kv_heads"], HD, case["page"], nv.KV_I8 if case["fmt"] == "i8" else nv.KV_E4M3,
                           0 if case["rope"] == "pairs" else 1)
        rope = case["rope"] != "none"
        cache = nv.Q8Cache(shape=shape, layer=0, nb=state["codes"][0].shape[0], pool_k=state["codes"][0].data_ptr(),
                           pool_v=state["codes"][1].data_ptr(), scale_k=state["scales"][0].data_ptr(), scale_v=state["scales"][1].data_ptr(),
                           tables=state["tables"].data_ptr(), table_stride=state["tables"].shape[1], slice_ids=state["slices"].data_ptr(),
                           rope_cs=state["cos"].data_ptr() if rope else None, rope_sn=state["sin"].data_ptr() if rope else None,
                           rope_rows=state["cos"].shape[0] if rope else 0, status=None)
        rows = nv.Q8Rows(n_sessions=case["sessions"], n_tokens=state["rows"], max_tokens=state["longest"],
                         io_dtype={"f32": nv.IO_F32, "f16": nv.IO_F16, "bf16": nv.IO_BF16}[case["io"]], n_past=state["past"].data_ptr(),
                         tok_start=None if state["uniform"] else state["start"].data_ptr(), q_stride=state["q"].stride(0),
                         k_stride=state["k"].stride(0), v_stride=state["v"].stride(0), out_stride=0)
        work = torch.empty(max(16, nv.q8_workspace_bytes(shape, rows)), dtype=torch.uint8, device=state["q"].device)
        state["handle"] = nv, cache, rows, work
    return state["handle"]


def _call(state):
    nv, cache, rows, work = _handle(state)
    op, stream = state["case"]["op"], torch.cuda.current_stream().cuda_stream
    if op in ("store", "read"):
        back = state["back"]
        if op == "store":
            nv.q8_append(cache, rows, state["k"].data_ptr(), state["v"].data_ptr(), stream)
        nv.q8_read(cache, rows, back[0].data_ptr(), back[1].data_ptr(), stream)
        return back
    nv.q8_append_attn(cache, rows, state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(), state["out"].data_ptr(),
                      state["case"]["window"], work.data_ptr(), work.numel(), stream)
    return state["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        got = _call(state)
    elif op == "read":
        got = _read(state)
    elif op == "store":
        _append(state)
        got = _read(state)
    else:
        _append(state)
        got = _attend(state)
    if op == "read":
        return {"k": got[0], "v": got[1]}
    cache = {"codes": state["codes"], "scales": state["scales"]}
    if op == "store":
        return {"k": got[0], "v": got[1], "cache": cache}
    return {"out": got, "cache": cache}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    past, new = _lens(case)
    H, N, page, fmt, w = case["heads"], case["kv_heads"], case["page"], case["fmt"], case["window"]
    top = Q_MAX[fmt]
    codes = [c.view(torch.uint8) for c in state["codes"]]
    scales = [s.double() for s in state["scales"]]
    c64, s64 = state["cos"].double(), state["sin"].double()

    def turned(x, p0):
        x = x.double()
        if case["rope"] == "none":
            return x
        n = x.shape[0]
        z = torch.complex(c64[p0:p0 + n], s64[p0:p0 + n])[:, None]
        if case["rope"] == "neox":
            y = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * z
            return torch.cat((y.real, y.imag), -1)
        return torch.view_as_real(torch.view_as_complex(x.reshape(n, -1, 64, 2).contiguous()) * z).reshape(x.shape)

    outs, at = [[], []], 0
    for s, (p, n) in enumerate(zip(past, new)):
        if not n:
            continue
        table = state["tables"][int(state["slices"][s])].long()
        first = max(0, p - w + 1) if w else 0
        lo = p if case["op"] in ("store", "read") else first
        pos = torch.arange(lo, p + n, device=table.device)
        phys, slot = table[pos // page], pos % page
        kv = []
        for i in (0, 1):
            x = codes[i][phys, slot].view(state["codes"][i].dtype).double() * scales[i][phys, :, slot][..., None]
            if case["op"] != "read":
                fresh = turned(state["k"][at:at + n], p) if i == 0 else state["v"][at:at + n].double()
                amax = fresh.abs().amax(-1, keepdim=True).clamp_min(MIN_AMAX)
                y = fresh.float() * (torch.full_like(amax, top).float() / amax.float())       # the codes are defined by these two fp32 operations
                y = y.round() if fmt == "i8" else y.to(torch.float8_e4m3fn)
                x[p - lo:] = y.double() * (amax / top)
            kv.append(x)
        if case["op"] in ("store", "read"):
            for i in (0, 1):
                outs[i].append(kv[i])
        else:
            q = turned(state["q"][at:at + n], p)
            here = torch.arange(p, p + n, device=table.device)
            seen = pos[None] <= here[:, None]
            if w:
                seen = seen & (pos[None] > here[:, None] - w)
            o = torch.empty(n, H, HD, dtype=torch.float64, device=table.device)
            for h in range(H):
                score = (q[:, h] @ kv[0][:, h // (H // N)].T) * HD ** -0.5
                o[:, h] = torch.softmax(score.masked_fill(~seen, -math.inf), -1) @ kv[1][:, h // (H // N)]
            outs[0].append(o)
        at += n
    if case["op"] in ("store", "read"):
        got = {"k": torch.cat(outs[0]), "v": torch.cat(outs[1])}
        return got if case["op"] == "read" else dict(got, cache=None)
    return {"out": torch.cat(outs[0]), "cache": None}
