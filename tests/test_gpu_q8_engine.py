"""Engines whose pools are 8-bit: the batch calls (prefill, append, attention, whole steps, graphs, host buffers), copy-on-write and
shared prefixes, against the plain 64-bit forms (q8_plain.py) applied to what the pools held before each step."""
import numpy as np
import pytest
import torch

from q8_plain import HD, Cache, attention_bound

pytestmark = pytest.mark.gpu


class Run:
    """An engine with a batch over all its sessions, and one step's inputs."""

    def __init__(self, nv, fmt, heads, kv_heads, past, *, page=16, neox=1, layers=2, ctx=256, spare=0, seed=5):
        self.nv, self.fmt, self.H, self.N, self.L, self.page, self.neox = nv, fmt, heads, kv_heads, layers, page, neox
        self.rng, self.stream = np.random.default_rng(seed), nv.Stream()
        self.eng = nv.Engine(layers, heads, kv_heads, ctx=ctx, n_slices=len(past) + spare, kv_block=page, rope_neox=neox,
                             kv_dtype=nv.KV_I8 if fmt == "i8" else nv.KV_E4M3)
        self.cs, self.sn = (torch.from_numpy(x.copy()) for x in self.eng.rope_tables())
        self.ss = [self.eng.session_create() for _ in past]
        for s in self.ss:
            self.eng.permute_pages(s, self.rng.permutation(self.eng.nblocks))
        for s, p in zip(self.ss, past):              # contexts of different lengths: one batch and one prefill each
            if p:
                b = self.eng.batch([s])
                self.prefill(b, p, check=False)
                b.close()

    def pools(self):
        nv = self.nv
        nv.check(nv.lib.dev_sync())
        codes = [torch.from_numpy(np.ascontiguousarray(x).view(np.uint8).copy()) for x in self.eng.read_pools()]
        return codes, [torch.from_numpy(x.copy()) for x in self.eng.read_scales()]

    def inputs(self, b, n=1):
        T = b.n * n
        return [self.rng.standard_normal((self.L, T, h, HD)).astype(np.float32) for h in (self.H, self.N, self.N)]

    def cases(self, b, x, n, pools):
        """The plain forms of one step: per layer a Cache over what the pools held before it."""
        past = [self.eng.n_past(s) for s in b.sessions]
        for layer in range(self.L):
            c = Cache(past, [n] * b.n, self.H, self.N, self.page, self.fmt, "f32", rope="neox" if self.neox else "pairs", poison=False)
            c.layer, (c.codes, c.scales), c.cs, c.sn = layer, pools, self.cs, self.sn
            c.slices = torch.arange(b.n)
            c.tables = torch.stack([torch.from_numpy(self.eng.pool.table(self.eng.session_slice(s)).astype(np.int32)) for s in b.sessions])
            c.q, c.k, c.v = (torch.from_numpy(t[layer]) for t in x)
            yield c

    def check(self, b, x, n, pools, out, window=0):
        """out [layers][rows][heads][128] of a step; pools (before it) take the step's rows."""
        assert b.device_status() == 0
        cases = list(self.cases(b, x, n, pools))
        for c in cases:
            c.append()
        now = self.pools()
        for want, got in zip(pools[0] + pools[1], now[0] + now[1]):
            assert bool((want.view(torch.uint8) == got.view(torch.uint8)).all()), "pools"
        for c in cases:
            c.window = window
            o, a, spread, floor = c.attend()
            got = torch.from_numpy(out[c.layer]).double()
            bound = attention_bound(c, o, a, spread, floor, False)         # q and the weights are rounded to fp16, by the header's word
            assert bool(torch.isfinite(got).all()) and bool(((got - o).abs() <= bound).all()), float(((got - o).abs() / bound).max())

    def prefill(self, b, n, check=True, window=0):
        nv = self.nv
        x = self.inputs(b, n)
        out = np.empty((self.L, b.n * n, self.H, HD), np.float32)
        pools = None
        for layer in range(self.L):
            q, k, v = (nv.to_device(t[layer]) for t in x)
            o = nv.DevBuf(out[layer].nbytes)
            if check and not layer:
                pools = self.pools()
            b.prefill(layer, n, q.ptr, k.ptr, v.ptr, o.ptr)
            nv.check(nv.lib.dev_sync())
            out[layer] = o.download(np.float32).reshape(out[layer].shape)
        if check:
            self.check(b, x, n, pools, out, window)
        assert b.device_status() == 0
        b.advance_by(n)

    def step(self, b, how, pools=None, window=0):
        """One decode step of all layers, by one of the ways the framework offers."""
        nv = self.nv
        pools = pools or self.pools()
        x = self.inputs(b)
        out = np.full((self.L, b.n, self.H, HD), 7, np.float32)
        if how.startswith("host"):
            # (this call advances the batch; the plain forms want the positions before it)
            q, k, v = (t.copy() for t in x)
            b.decode_step_host(q.ctypes.data, k.ctypes.data, v.ctypes.data, out.ctypes.data, per_layer=int(how[-1]))
            past = [self.eng.n_past(s) - 1 for s in b.sessions]
        else:
            q, k, v = (nv.to_device(t) for t in x)
            o = nv.DevBuf(out.nbytes)
            nq, nk = b.n * self.H * HD * 4, b.n * self.N * HD * 4
            if how.startswith("run"):
                b.run_steps(1, q.ptr, k.ptr, v.ptr, o.ptr, 0, 0, int(how[-1]), self.stream.h)
                self.stream.sync()
                past = [self.eng.n_past(s) - 1 for s in b.sessions]
            else:
                past = None
                if how == "all":
                    b.step_all_layers(q.ptr, k.ptr, v.ptr, o.ptr)
                elif how == "layers":
                    b.append_layers(0, self.L, q.ptr, k.ptr, v.ptr)
                else:
                    for i in range(self.L):
                        at = (q.ptr + i * nq, k.ptr + i * nk, v.ptr + i * nk)
                        if how == "both":
                            b.append_attn(i, *at, o.ptr + i * nq)
                        else:
                            b.append(i, *at)
                            b.attn(i, q.ptr + i * nq, o.ptr + i * nq)
                if how == "layers":
                    for i in range(self.L):
                        b.attn(i, q.ptr + i * nq, o.ptr + i * nq)
            nv.check(nv.lib.dev_sync())
            out = o.download(np.float32).reshape(out.shape)
            if not how.startswith("run"):            # k is rotated in place whichever way was taken (runs in a graph use copies)
                got = k.download(np.float32).reshape(x[1].shape)
                from q8_plain import rotate
                for i, c in enumerate(self.cases(b, x, 1, pools)):
                    want = rotate(c.k, c.positions(), self.cs, self.sn, c.rope)
                    assert bool((torch.from_numpy(got[i]).view(torch.int32) == want.view(torch.int32)).all()), "k in place"
        if past is None:
            self.check(b, x, 1, pools, out)
            b.advance()
        else:
            for s, p in zip(b.sessions, past):
                self.eng.set_n_past(s, p)
            self.check(b, x, 1, pools, out)
            for s, p in zip(b.sessions, past):
                self.eng.set_n_past(s, p + 1)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,page,neox", [(28, 4, 16, 1), (6, 2, 8, 0), (4, 1, 64, 1), (24, 2, 32, 1), (3, 3, 16, 0)])
def test_every_way_of_a_step(nv, fmt, heads, kv_heads, page, neox):
    r = Run(nv, fmt, heads, kv_heads, [0, 30, 7], page=page, neox=neox)
    b = r.eng.batch(r.ss)
    assert nv.lib.nova_batch_get_kernel(b.h) == 1
    r.prefill(b, 21)
    r.prefill(b, 1)
    for fused in (0, 1):
        b.set_fused_append(fused)
        for how in ("apart", "both", "all", "layers", "run0", "run1", "run2", "run2", "host0", "host1"):
            r.step(b, how)
    r.prefill(b, 40)
    b.close()
    r.eng.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_windowed_prefill(nv, fmt):
    r = Run(nv, fmt, 12, 2, [50, 3])
    b = r.eng.batch(r.ss)
    b.set_window(20)
    r.prefill(b, 33, window=20)
    r.prefill(b, 1, window=20)
    b.set_window(0)
    r.step(b, "both")
    b.close()
    r.eng.close()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("page", [8, 16])
def test_shared_prefix_is_copied_on_write_with_its_scales(nv, fmt, page):
    r = Run(nv, fmt, 14, 2, [37], page=page, spare=5)
    donor = r.ss[0]
    *forks, late = [r.eng.session_create() for _ in range(4)]
    for f in forks + [late]:
        r.eng.attach_prefix(f, donor, 37)
    before = r.pools()
    tail = int(r.eng.pool.table(r.eng.session_slice(donor))[36 // page])
    b = r.eng.batch(forks)
    assert b.cow() == 3
    now = r.pools()
    for f in forks:                 # the copies hold the donor's codes and scales in all layers
        mine = int(r.eng.pool.table(r.eng.session_slice(f))[36 // page])
        assert mine != tail
        for x in now[0] + now[1]:
            assert bool((x[:, mine].view(torch.uint8) == x[:, tail].view(torch.uint8)).all())
    r.step(b, "both")
    assert b.cow() == 0
    r.step(b, "run1")
    r.prefill(b, 9)
    after = r.pools()
    for x, y in zip(before[0] + before[1], after[0] + after[1]):
        assert bool((x[:, tail].view(torch.uint8) == y[:, tail].view(torch.uint8)).all()), "the donor's page"
    b.close()
    # a prefill un-shares the pages it lands in by itself
    b = r.eng.batch([late])
    x = r.inputs(b, 5)
    q, k, v = (nv.to_device(t[0]) for t in x)
    o = nv.DevBuf(x[0][0].nbytes)
    b.prefill(0, 5, q.ptr, k.ptr, v.ptr, o.ptr)
    nv.check(nv.lib.dev_sync())
    assert int(r.eng.pool.table(r.eng.session_slice(late))[36 // page]) != tail and b.device_status() == 0
    assert bool((r.pools()[1][0][:, tail] == before[1][0][:, tail]).all())
    b.close()
    r.eng.close()


def test_new_sessions_find_empty_pages(nv):
    r = Run(nv, "i8", 4, 2, [60])
    r.eng.session_destroy(r.ss[0])
    s = r.eng.session_create()
    codes, scales = r.pools()
    for x in codes + scales:
        assert bool((x[:, r.eng.pool.table(r.eng.session_slice(s)).tolist()] == 0).all())
    r.eng.close()


def test_operators_on_an_engines_cache(nv):
    """The operators of the 8-bit section on an engine's own pools: bf16 rows of several sessions at once."""
    r = Run(nv, "e4m3", 8, 2, [0, 40, 11])
    new = [5, 0, 17]
    T = sum(new)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, HD, generator=g).bfloat16() for h in (8, 2, 2))
    pools = r.pools()
    past = torch.tensor([r.eng.n_past(s) for s in r.ss], dtype=torch.int32)
    start = torch.tensor([0, 5, 5, 22], dtype=torch.int32)
    slices = torch.tensor([r.eng.session_slice(s) for s in r.ss], dtype=torch.int32)
    dev = [t.cuda() for t in (q, k, v, past, start, slices)]
    c = Cache(past.tolist(), new, 8, 2, 16, "e4m3", "bf16", poison=False)
    c.layer, (c.codes, c.scales), c.cs, c.sn, c.slices = 1, pools, r.cs, r.sn, slices
    c.tables = torch.stack([torch.from_numpy(r.eng.pool.table(i).astype(np.int32)) for i in range(r.eng.desc.n_slices)])
    c.q, c.k, c.v = q, k, v
    cache = r.eng.q8_cache(1)
    cache.slice_ids = dev[5].data_ptr()
    rows = nv.Q8Rows(3, T, 17, nv.IO_BF16, dev[3].data_ptr(), dev[4].data_ptr())
    out = torch.zeros(T, 8, HD, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(nv.q8_workspace_bytes(cache.shape, rows), dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    nv.q8_append_attn(cache, rows, dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), out.data_ptr(), 0, work.data_ptr(), work.numel(), s)
    torch.cuda.synchronize()
    c.append()
    now = r.pools()
    for want, got in zip(pools[0] + pools[1], now[0] + now[1]):
        assert bool((want.view(torch.uint8) == got.view(torch.uint8)).all())
    o, a, spread, floor = c.attend()
    off = (out.cpu().double() - o).abs()
    assert bool((off <= attention_bound(c, o, a, spread, floor, False)).all())
    r.eng.close()


def test_workload_fills_and_steps(nv):
    from conflux_nova_b200.workloads import Workload
    w = Workload("qwen25_1p5b", [100, 33], seed=3, steps=4, n_layers=2, kv_dtype=nv.KV_I8)
    dq, dk, dv = w.device_step_inputs(0)
    out = nv.DevBuf(w.step_input_sizes()[0] * 4)
    w.batch.run_steps(2, dq.ptr, dk.ptr, dv.ptr, out.ptr, 0, 0, 1)
    nv.check(nv.lib.dev_sync())
    assert w.batch.device_status() == 0
    assert w.kv_bytes_per_step([99, 32]) == (133 + 2) * 2 * 2 * 132 * 2
    assert np.isfinite(out.download(np.float32)).all()
    w.close()


def test_refusals(nv):
    r = Run(nv, "i8", 8, 2, [20, 20], spare=1)
    b = r.eng.batch(r.ss)
    lib, U, I = nv.lib, nv.ERR_UNSUPPORTED, nv.ERR_INVALID
    x = nv.DevBuf(1 << 16)
    assert lib.nova_batch_set_kernel(b.h, 0) == U and lib.nova_batch_set_kernel(b.h, 1) == nv.OK
    assert lib.nova_batch_set_prefill_kernel(b.h, 0) == U and lib.nova_batch_set_cascade(b.h, 1) == U
    assert lib.nova_batch_attn_partial(b.h, 0, x.ptr, 0, 1, x.ptr, None) == U
    assert lib.nova_batch_attn_partial_layers(b.h, 0, 1, x.ptr, 0, 1, x.ptr, None) == U
    assert lib.nova_batch_append(b.h, 0, x.ptr + 4, x.ptr, x.ptr, None) == I and lib.nova_batch_attn(b.h, 0, x.ptr, x.ptr + 8, None) == I
    assert lib.nova_batch_prefill(b.h, 0, 8193, x.ptr, x.ptr, x.ptr, x.ptr, None) == nv.ERR_TOO_LARGE
    sh, c = r.eng.shape(), nv.Q8Cache()
    tab = lib.nova_kv_table_slot(r.eng.h, 0)
    import ctypes as C
    for which in (0, 1):
        lib.nova_launcher_set_kernel(which)
        assert lib.nova_launch_attn_decode_paged(C.byref(sh), x.ptr, r.eng.k_base, r.eng.v_base, tab, 0, r.eng.nb, 5, x.ptr, x.ptr, None) == U
    lib.nova_launcher_set_kernel(0)
    assert lib.nova_launch_attn_decode_paged_static(C.byref(sh), x.ptr, r.eng.k_base, r.eng.v_base, tab, 0, r.eng.nb, 5, x.ptr, None) == U
    assert lib.nova_launch_rope_append_paged(C.byref(sh), r.eng.k_base, r.eng.v_base, tab, 0, r.eng.nb, 1, 0, x.ptr, x.ptr, x.ptr,
                                             lib.nova_rope_cos(r.eng.h), lib.nova_rope_sin(r.eng.h), None) == U
    assert lib.nova_engine_q8_cache(r.eng.h, 2, C.byref(c)) == I and lib.nova_engine_q8_cache(r.eng.h, 0, None) == I
    r.step(b, "both")
    b.close()
    r.eng.close()
    plain = nv.Engine(1, 8, 2, ctx=64, n_slices=1)
    assert lib.nova_engine_q8_cache(plain.h, 0, C.byref(c)) == U
    plain.close()
    assert lib.nova_engine_create(C.byref(nv.EngineDesc(1, 4 * 129, 4, 128, 16, nv.KV_I8, 10000, 1, 1, 1, 64, 64, 0, 1)), C.byref(C.c_void_p())) == U
