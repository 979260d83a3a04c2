"""Plain 64-bit forms of the 8-bit paged cache's operators and the cases that its tests run (CPU torch, loops)."""
import math

import torch

HD = 128
QMAX = {"i8": 127.0, "e4m3": 448.0}
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MIN_AMAX = 2.0 ** -60


def rope_tables(rows, theta=1e6):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * torch.exp(torch.arange(64, dtype=torch.float64) * (-math.log(theta) / 64))
    return ang.cos().float(), ang.sin().float()


def rotate(x, pos, cs, sn, kind):
    """x [n][heads][128] fp32; the pair (a, b) becomes (fma(a, c, -rn(b s)), fma(a, s, rn(b c))), rounded to fp32 once each.
    In 64 bits the product a*c is exact and the sum is rounded to 53 bits before the 24: the same value but for ties that need
    more than 53 bits."""
    if kind == "none":
        return x.float()
    x = x.float()
    c, s = cs[pos][:, None], sn[pos][:, None]
    a, b = (x[..., :64], x[..., 64:]) if kind == "neox" else (x[..., 0::2], x[..., 1::2])
    u = (a.double() * c.double() - (b * s).double()).float()
    w = (a.double() * s.double() + (b * c).double()).float()
    return torch.cat((u, w), -1) if kind == "neox" else torch.stack((u, w), -1).flatten(-2)


def quantise(x, fmt):
    """fp32 rows [..., 128] -> codes (as a torch tensor of the format) and scales."""
    amax = x.abs().amax(-1).clamp_min(MIN_AMAX)
    q = torch.full_like(amax, QMAX[fmt])        # tensors on both sides: a scalar over a tensor would go through a rounded reciprocal
    y = x * (q / amax)[..., None]
    return (y.round().to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn)), amax / q


class Cache:
    """Codes, scales, tables of a few sessions on the CPU; `device()` puts them on the GPU behind the descriptors."""

    def __init__(self, past, new, heads, kv_heads, page, fmt, io, *, rope="neox", packed=False, seed=0, layers=2, layer=1, window=0,
                 poison=True, uniform=False, scale_spread=0.5, q_gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.past, self.new, self.H, self.N, self.page, self.fmt, self.io = list(past), list(new), heads, kv_heads, page, fmt, io
        self.rope, self.window, self.layer, self.uniform = rope, window, layer, uniform
        S = len(past)
        need = [(p + n + page - 1) // page for p, n in zip(past, new)]
        self.nb = sum(need) + 2
        width = max(need + [0]) + 1
        order = torch.randperm(self.nb, generator=g)
        self.slices = torch.randperm(S, generator=g).to(torch.int32)
        self.tables = torch.full((S, width), -1, dtype=torch.int32)
        at = 0
        for s, c in enumerate(need):
            self.tables[int(self.slices[s]), :c] = order[at:at + c].to(torch.int32)
            at += c
        shape = (layers, self.nb, page, kv_heads, HD)
        bad = 0x7f                                   # 127, or the e4m3 NaN: what nobody may look at
        self.codes, self.scales = [], []
        for _ in range(2):
            if fmt == "i8":
                c = (torch.randn(shape, generator=g) * 47).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
            else:
                c = (torch.randn(shape, generator=g) * 166).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            sc = torch.exp(torch.randn(layers, self.nb, kv_heads, page, generator=g) * scale_spread) / (47 if fmt == "i8" else 166)
            if poison:
                keep_c, keep_s = torch.full_like(c, bad), torch.full_like(sc, math.nan)
                for s, p in enumerate(past):
                    for j in range(p):
                        ph = int(self.tables[int(self.slices[s]), j // page])
                        keep_c[:, ph, j % page] = c[:, ph, j % page]
                        keep_s[:, ph, :, j % page] = sc[:, ph, :, j % page]
                c, sc = keep_c, keep_s
            self.codes.append(c)
            self.scales.append(sc)
        T = sum(new)
        qkv = (torch.randn(T, heads + 2 * kv_heads, HD, generator=g) * q_gain).to(IO[io])
        self.qkv = qkv
        self.q, self.k, self.v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        self.packed = packed
        self.cs, self.sn = rope_tables(max([p + n for p, n in zip(past, new)] + [0]) + 1)
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)

    # ---- plain forms
    def typed(self, c):
        return c.view(torch.int8 if self.fmt == "i8" else torch.float8_e4m3fn)

    def place(self, s, j):
        return int(self.tables[int(self.slices[s]), j // self.page]), j % self.page

    def positions(self):
        return torch.tensor([p + t for p, n in zip(self.past, self.new) for t in range(n)], dtype=torch.long)

    def append(self):
        """Writes the new rows into the CPU copy."""
        pos = self.positions()
        rows = (rotate(self.k, pos, self.cs, self.sn, self.rope), self.v.float())
        for i in (0, 1):
            c, sc = quantise(rows[i], self.fmt)
            at = 0
            for s, (p, n) in enumerate(zip(self.past, self.new)):
                for t in range(n):
                    ph, slot = self.place(s, p + t)
                    self.codes[i][self.layer, ph, slot] = c.view(torch.uint8)[at]
                    self.scales[i][self.layer, ph, :, slot] = sc[at]
                    at += 1

    def values(self, i, s, lo, hi):
        """[hi - lo][N][128] of session s in 64 bits, and in fp32 (one rounded product)."""
        if hi <= lo:
            z = torch.zeros(0, self.N, HD)
            return z.double(), z
        j = torch.arange(lo, hi)
        ph, slot = self.tables[int(self.slices[s])].long()[j // self.page], j % self.page
        c = self.typed(self.codes[i][self.layer][ph, slot]).float()
        sc = self.scales[i][self.layer][ph, :, slot][..., None]
        return c.double() * sc.double(), c * sc

    def read(self):
        parts = [[self.values(i, s, p, p + n)[1] for s, (p, n) in enumerate(zip(self.past, self.new))] for i in (0, 1)]
        return [torch.cat(x).to(IO[self.io]) for x in parts]

    def attend(self):
        """(o, a, spread, floor): the outputs in 64 bits, the sum of weights times |v|, per row the largest sum of |q k| / sqrt(128), and
        the sum of |codes of v| times the row's largest weight (p times v's scale)."""
        o = torch.zeros(sum(self.new), self.H, HD, dtype=torch.float64)
        a, spread, floor = o.clone(), torch.zeros(sum(self.new), self.H, dtype=torch.float64), o.clone()
        pos = self.positions()
        q = rotate(self.q, pos, self.cs, self.sn, self.rope).double()
        G, at = self.H // self.N, 0
        for s, (p, n) in enumerate(zip(self.past, self.new)):
            if not n:
                continue
            k, v = self.values(0, s, 0, p + n)[0], self.values(1, s, 0, p + n)[0]
            key, here = torch.arange(p + n)[None], torch.arange(p, p + n)[:, None]
            seen = key <= here
            if self.window:
                seen &= key > here - self.window
            for h in range(self.H):
                kh, vh, qh = k[:, h // G], v[:, h // G], q[at:at + n, h]
                score = (qh @ kh.T) * HD ** -0.5
                w = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
                o[at:at + n, h] = w @ vh
                a[at:at + n, h] = w @ vh.abs()
                j = torch.arange(p + n)
                ph, slot = self.tables[int(self.slices[s])].long()[j // self.page], j % self.page
                sv = self.scales[1][self.layer][ph, h // G, slot].double()
                floor[at:at + n, h] = (w * sv).amax(-1, keepdim=True) * (seen.double() @ (vh / sv[:, None]).abs())
                spread[at:at + n, h] = ((qh.abs() @ kh.abs().T) * HD ** -0.5).masked_fill(~seen, 0).amax(-1)
            at += n
        return o, a, spread, floor

    # ---- the framework's side
    def device(self, nv, dev="cuda", extra_rows=0, status=True):
        """Uploads; extra_rows more rows of q / k / v / out behind the last session's."""
        d = {"codes": [c.clone().to(dev) for c in self.codes], "scales": [s.clone().to(dev) for s in self.scales],
             "tables": self.tables.to(dev), "slices": self.slices.to(dev), "cs": self.cs.to(dev), "sn": self.sn.to(dev),
             "past": torch.tensor(self.past, dtype=torch.int32, device=dev), "start": torch.tensor(self.start, dtype=torch.int32, device=dev),
             "status": torch.zeros(1, dtype=torch.int32, device=dev)}
        qkv = self.qkv
        if extra_rows:
            qkv = torch.cat((qkv, torch.full((extra_rows,) + tuple(qkv.shape[1:]), math.nan, dtype=qkv.dtype)))
        qkv = qkv.to(dev)
        H, N = self.H, self.N
        d["qkv"] = qkv
        d["q"], d["k"], d["v"] = qkv[:, :H], qkv[:, H:H + N], qkv[:, H + N:]
        if not self.packed:
            d["q"], d["k"], d["v"] = (d[x].contiguous() for x in "qkv")
        T = qkv.shape[0]
        d["out"] = torch.full((T, H, HD), 7.0, dtype=IO[self.io], device=dev)
        d["back"] = [torch.full((T, N, HD), 7.0, dtype=IO[self.io], device=dev) for _ in range(2)]
        shape = nv.KvShape(H, N, HD, self.page, nv.KV_I8 if self.fmt == "i8" else nv.KV_E4M3, 0 if self.rope == "pairs" else 1)
        rope = self.rope != "none"
        d["cache"] = nv.Q8Cache(shape=shape, layer=self.layer, nb=self.nb, pool_k=d["codes"][0].data_ptr(), pool_v=d["codes"][1].data_ptr(),
                                scale_k=d["scales"][0].data_ptr(), scale_v=d["scales"][1].data_ptr(), tables=d["tables"].data_ptr(),
                                table_stride=self.tables.shape[1], slice_ids=d["slices"].data_ptr(), rope_cs=d["cs"].data_ptr() if rope else None,
                                rope_sn=d["sn"].data_ptr() if rope else None, rope_rows=self.cs.shape[0] if rope else 0,
                                status=d["status"].data_ptr() if status else None)
        d["rows"] = nv.Q8Rows(n_sessions=len(self.past), n_tokens=sum(self.new) if self.uniform else T, max_tokens=max(self.new), io_dtype={"f32": nv.IO_F32, "f16": nv.IO_F16, "bf16": nv.IO_BF16}[self.io],
                              n_past=d["past"].data_ptr(), tok_start=None if self.uniform else d["start"].data_ptr(), q_stride=d["q"].stride(0) if T else 0,
                              k_stride=d["k"].stride(0) if T else 0, v_stride=d["v"].stride(0) if T else 0, out_stride=0)
        d["work"] = torch.empty(max(16, nv.q8_workspace_bytes(shape, d["rows"])), dtype=torch.uint8, device=dev)
        return d


def call(nv, d, what, window=0, stream=None):
    """One operator on the device side of a Cache."""
    stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
    c, r = d["cache"], d["rows"]
    if what == "append":
        nv.q8_append(c, r, d["k"].data_ptr(), d["v"].data_ptr(), stream)
    elif what == "read":
        nv.q8_read(c, r, d["back"][0].data_ptr(), d["back"][1].data_ptr(), stream)
    elif what == "attn":
        nv.q8_attn(c, r, d["q"].data_ptr(), d["out"].data_ptr(), window, d["work"].data_ptr(), d["work"].numel(), stream)
    else:
        nv.q8_append_attn(c, r, d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), d["out"].data_ptr(), window, d["work"].data_ptr(),
                          d["work"].numel(), stream)


def attention_bound(case, o, a, spread, floor, exact_q):
    """How far an output may be off.
    One step of the sum: weights p = exp(s), so a score off by e takes p off by e (1 + e) and the quotient off by 2 e at most,
    relative to a = sum p |v|.  Scores: q goes to fp16 (2^-11 relative, exact_q: fp16 hi + lo, 2^-21), in chunks K too (2^-11 for the
    product, 2^-14 for a scale whose second part is subnormal), which moves a score by at most that times spread = sum |q k| / sqrt(128); the fp32 accumulation of 128 products by 2^-19 times spread (17 additions rounded or
    truncated to 24 bits), the exponential's argument by 2^-23 of a magnitude below 2 spread.  Weights go to fp16 (2^-11; hi + lo: 2^-21),
    in chunks V too (2^-11 for its scale, 2^-11 for the product; below fp16's normal range 2^-25),
    their sums are rounded once per 16 keys (2^-23 each).  A weight below fp16's normal range is off by 2^-25 whatever it is, and
    the largest weight of a row (p times v's scale) goes in as 2^11 or more, in chunks 2^7: floor 2^-36, 2^-32 in all.  Last the rounding of the output
    itself, half a step."""
    keys = max([p + n for p, n in zip(case.past, case.new)] + [1])
    chunk = max(case.new) > 1 or case.H // case.N > 8
    q_err, p_err = (2.0 ** -21, 2.0 ** -21) if exact_q else (2.0 ** -11, 2.0 ** -11)
    if chunk:
        q_err, p_err = q_err + 2.0 ** -11 + 2.0 ** -14, p_err + 2 * 2.0 ** -11
    e = spread * (q_err + 2.0 ** -19 + 2.0 ** -22)
    rel = 2 * (e * (1 + e) + p_err) + (keys / 16 + 64) * 2.0 ** -23
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[case.io]
    tiny = {"f32": 1e-37, "f16": 2.0 ** -25, "bf16": 1e-37}[case.io]
    return a * rel[..., None] + floor * 2.0 ** (-32 if chunk else -36) + o.abs() * half + tiny + (2.0 ** -25 if chunk else 0.0)
