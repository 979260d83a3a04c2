"""How the 8-bit cache operators are called: the first call of a process within a capture, calls of several host threads at once."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from conftest import ROOT
from q8_plain import Cache, call
from test_gpu_q8 import check_cache, check_out

pytestmark = pytest.mark.gpu

CASES = {"decode": ([50, 10, 90], [1, 1, 1], "f16"), "chunk": ([50, 10, 90], [3, 0, 20], "bf16")}


def capture_first(kind):
    """(in a process of its own) No call of the library before the captured one."""
    import __graft_entry__ as g
    nv = g.load_package()
    past, new, io = CASES[kind]
    case = Cache(past, new, 14, 2, 16, "i8", io)
    d = case.device(nv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(nv, d, "append_attn")
        call(nv, d, "read")
    torch.cuda.synchronize()
    assert bool((d["out"] == 7).all())
    graph.replay()
    torch.cuda.synchronize()
    case.append()
    check_cache(case, d)
    check_out(case, d)


@pytest.mark.parametrize("kind", list(CASES))
def test_the_first_call_may_be_captured(nv, kind):
    code = f"import sys; sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]; import test_gpu_q8_calls as t; t.capture_first({kind!r})"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


def test_threads_that_call_at_once(nv):
    """Four host threads, each with its own stream, cache and workspace (and a status word that all share)."""
    cases = [Cache([300 + i, 10, 90], [1, 1, 1] if i % 2 else [9, 0, 20], 14, 2, 16, "e4m3" if i < 2 else "i8", "bf16", seed=i) for i in range(4)]
    ds = [c.device(nv) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for d in ds:
        d["cache"].status = ds[0]["status"].data_ptr()
    torch.cuda.synchronize()
    failed = []

    def work(d, s):
        try:
            for _ in range(20):
                call(nv, d, "append_attn", stream=s.cuda_stream)
                call(nv, d, "read", stream=s.cuda_stream)
        except Exception as e:                               # pragma: no cover
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(ds, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and int(ds[0]["status"]) == 0
    for case, d in zip(cases, ds):
        case.append()
        check_cache(case, d)
        check_out(case, d)
