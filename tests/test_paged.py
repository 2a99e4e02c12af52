"""The paged cache without a GPU: the C ABI's structures and refusals, and the oracle against
the sliding-window oracle."""
from __future__ import annotations

import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

from oracle import paged as op
from oracle import swa as oswa
from tests.conftest import ROOT

FAKE = 1 << 20  # 16-byte aligned, never dereferenced


@pytest.fixture(scope="module")
def capi():
    from pseudobrain_b200 import build
    build.build()
    from pseudobrain_b200 import _capi
    return _capi


@pytest.mark.parametrize("cname,pyname", [("pbk_paged_cache", "PbkPagedCache"), ("pbk_paged_batch", "PbkPagedBatch"),
                                          ("pbk_paged_attend_desc", "PbkPagedAttendDesc"),
                                          ("pbk_paged_observe_desc", "PbkPagedObserveDesc")])
def test_descriptor_layout_matches_header(capi, cname, pyname):
    cls = getattr(capi, pyname)
    fields = [f for f, _ in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"pbk.h\"\nint main(void){\n"
    src += "".join(f'printf("%zu\\n", offsetof({cname}, {f}));\n' for f in fields)
    src += f'printf("%zu\\n", sizeof({cname})); return 0; }}\n'
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        with open(c, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(cls, f).offset for f in fields] + [ctypes.sizeof(cls)]


def _cache(capi, **over):
    f = dict(kv=2, d=128, page=16, pages=10, dtype=capi.PBK_BF16, k_pages=FAKE, v_pages=FAKE, stride_page=4096,
             stride_head=2048, stride_entry=128, mass=FAKE, pos=FAKE, meta_page=32, meta_head=16)
    return capi.PbkPagedCache(**{**f, **over})


def _batch(capi, **over):
    return capi.PbkPagedBatch(**{**dict(batch=3, width=5, block_table=FAKE, table_stride=5, lengths=FAKE, seen=FAKE),
                                 **over})


def _attend(capi, **over):
    f = dict(h=8, window=0, sinks=0, accumulate=0, scale=0.1, out_dtype=capi.PBK_BF16, q=FAKE, q_stride_b=1024,
             q_stride_h=128, out=FAKE, out_stride_b=1024, out_stride_h=128, lse=FAKE)
    return capi.PbkPagedAttendDesc(**{**f, **over})


@pytest.mark.parametrize("where,over,status", [
    ("cache", {"page": 12}, "SHAPE"), ("cache", {"page": 4}, "SHAPE"), ("cache", {"page": 512}, "SHAPE"),
    ("cache", {"d": 96}, "SHAPE"), ("cache", {"dtype": 0}, "DTYPE"), ("cache", {"kv": 0}, "INVALID"),
    ("cache", {"kv": 3}, "SHAPE"), ("cache", {"k_pages": None}, "INVALID"), ("cache", {"v_pages": FAKE + 2}, "ALIGN"),
    ("cache", {"stride_entry": 130}, "ALIGN"), ("cache", {"stride_head": 0}, "INVALID"),
    ("cache", {"mass": FAKE + 4}, "ALIGN"), ("cache", {"meta_head": 18}, "ALIGN"), ("cache", {"kv": 65536}, "SHAPE"),
    ("batch", {"batch": -1}, "INVALID"), ("batch", {"batch": 65536}, "SHAPE"), ("batch", {"lengths": None}, "INVALID"),
    ("batch", {"block_table": None}, "INVALID"), ("batch", {"width": 1 << 28}, "SHAPE"),
    ("desc", {"h": 130}, "SHAPE"), ("desc", {"h": 0}, "INVALID"), ("desc", {"sinks": -1}, "INVALID"),
    ("desc", {"scale": 0.0}, "INVALID"), ("desc", {"scale": float("nan")}, "INVALID"),
    ("desc", {"out_dtype": 2}, "DTYPE"), ("desc", {"q": None}, "INVALID"), ("desc", {"lse": None}, "INVALID"),
    ("desc", {"q_stride_h": 129}, "ALIGN"), ("desc", {"out": FAKE + 4}, "ALIGN"),
])
def test_attend_refuses_on_the_host(capi, where, over, status):
    c, b, d = _cache(capi), _batch(capi), _attend(capi)
    for k, v in over.items():
        setattr({"cache": c, "batch": b, "desc": d}[where], k, v)
    want = getattr(capi, f"PBK_ERR_{status}")
    assert capi.LIB.pbk_paged_attend_workspace(c, b, d) == 0
    assert capi.LIB.pbk_paged_attend(c, b, d, FAKE, 1 << 40, None) == want


def test_the_other_calls_refuse_on_the_host(capi):
    L = capi.LIB
    c, b = _cache(capi), _batch(capi)
    o = capi.PbkPagedObserveDesc(8, 16, 0.1, 0, FAKE, 8192, 1024, 128)
    assert L.pbk_paged_observe(_cache(capi, mass=None), b, o, FAKE, 1 << 40, None) == capi.PBK_ERR_INVALID
    o.q_stride_t = 0
    assert L.pbk_paged_observe(c, b, o, FAKE, 1 << 40, None) == capi.PBK_ERR_INVALID  # one query's row for all
    o.queries, o.q_stride_t = 1025, 1024
    assert L.pbk_paged_observe(c, b, o, FAKE, 1 << 40, None) == capi.PBK_ERR_SHAPE
    assert L.pbk_paged_append(c, b, FAKE, FAKE, 256, 128, 4, None, None) == capi.PBK_ERR_INVALID  # 4 tokens, 3 sequences
    assert L.pbk_paged_append(c, b, FAKE, FAKE + 8, 256, 128, 3, None, None) == capi.PBK_ERR_ALIGN
    sel = lambda budget, recent, sinks, moves, cc=c, bb=b: L.pbk_paged_select(  # noqa: E731
        cc, bb, budget, recent, sinks, FAKE, FAKE, FAKE, moves, None)
    assert sel(32, 30, 3, 32) == capi.PBK_ERR_INVALID     # more protected than kept
    assert sel(0, 0, 0, 32) == capi.PBK_ERR_INVALID
    assert sel(32, 0, 0, 31) == capi.PBK_ERR_SHAPE        # capacity 80, budget 32: 32 moves
    assert sel(64, 0, 0, 15) == capi.PBK_ERR_SHAPE        # 16 moves
    assert sel(32, 0, 0, 32, _cache(capi, pos=None)) == capi.PBK_ERR_INVALID
    assert sel(32, 0, 0, 32, c, _batch(capi, width=(1 << 19) + 1)) == capi.PBK_ERR_SHAPE  # over 2^23 entries
    assert sel(32, 0, 0, 32, c, _batch(capi, seen=None)) == capi.PBK_ERR_INVALID
    assert L.pbk_paged_move(c, b, FAKE, None, FAKE, 3, None) == capi.PBK_ERR_INVALID
    none = _batch(capi, batch=0)
    assert L.pbk_paged_attend(c, none, _attend(capi), None, 0, None) == capi.PBK_OK
    assert L.pbk_paged_move(c, none, FAKE, FAKE, FAKE, 3, None) == capi.PBK_OK
    assert sel(32, 0, 0, 32, c, none) == capi.PBK_OK


def test_module_imports_and_refuses_cpu_tensors(capi):
    import torch
    from pseudobrain_b200 import paged_cache as P
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.PagedCache(torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (1, 0)])
def test_oracle_attention_is_the_last_row_of_the_window_oracle(window, sinks):
    rng = np.random.default_rng(0)
    b, h, kv, n, d, page = 2, 6, 2, 45, 64, 8
    k, v = rng.standard_normal((2, b, kv, n, d))
    q = rng.standard_normal((b, h, n, d))
    table = rng.permutation(b * 6).reshape(b, 6)
    kp, vp = np.full((2, b * 6, kv, page, d), np.nan)
    for i in range(b):
        p, r = op.entry(table, page, i, np.arange(n))
        kp[p, :, r], vp[p, :, r] = k[i].transpose(1, 0, 2), v[i].transpose(1, 0, 2)
    out, lse, w = op.attend(q[:, :, -1], kp, vp, table, [n, n], window, sinks)
    assert np.allclose(out, oswa.causal_attention(q, k, v, window, sinks)[:, :, -1], atol=1e-12)
    assert np.allclose([x.sum() for x in w], h)
    if window is None:
        assert np.allclose(op.observe(q[:, :, -1:].transpose(0, 2, 1, 3), kp, table, [n, n]), w, atol=1e-12)


def _host_cache(capi):
    """Host tensors in the place of the device's (their device index is -1), for what is decided in
    Python: (cache, q, table, lengths)."""
    import torch
    from pseudobrain_b200 import paged_cache as P
    cache = object.__new__(P.PagedCache)
    cache.k_pages = cache.v_pages = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    cache.mass, cache.pos = torch.zeros(4, 2, 16), None
    cache.device, cache._index, cache._only_gpu = torch.device("cpu"), -1, False
    cache._desc = _cache(capi, d=64)
    cache._ref = ctypes.byref(cache._desc)
    return (cache, torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 1, dtype=torch.int32),
            torch.zeros(3, dtype=torch.int32))


def test_workspaces_are_sized_on_the_caches_device(capi, monkeypatch):
    """A cache on another device than the current one: the workspace's size, which follows the
    device's SMs and clusters, and the launch are asked for with the cache's device current."""
    import contextlib
    import types

    import torch
    from pseudobrain_b200 import paged_cache as P
    here, seen = [3], []

    @contextlib.contextmanager
    def device(i):
        here[0], was = i, here[0]
        yield
        here[0] = was

    def size(*args):
        seen.append(("size", here[0]))
        return 256

    def launch(*args):
        seen.append(("launch", here[0]))
        return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: here[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(P, "LIB", types.SimpleNamespace(
        pbk_paged_attend=launch, pbk_paged_attend_workspace=size, pbk_paged_observe=launch, pbk_paged_observe_workspace=size))
    cache, q, table, lens = _host_cache(capi)
    P.paged_attend(cache, q, table, lens)
    P.paged_observe_(cache, q[:, None], table, lens)
    assert seen == [("size", -1), ("launch", -1)] * 2 and here == [3]


def test_attention_refuses_to_lose_a_gradient(capi, monkeypatch):
    """A query or a pool that requires grad is refused while gradients are recorded, not answered
    with a result that has none; without recording the call runs."""
    import types

    import torch
    from pseudobrain_b200 import paged_cache as P
    calls = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(P, "LIB", types.SimpleNamespace(pbk_paged_attend=lambda *a: calls.append(a) or 0,
                                                        pbk_paged_attend_workspace=lambda *a: 0))
    cache, q, table, lens = _host_cache(capi)
    with pytest.raises(RuntimeError, match="no backward pass"):
        P.paged_attend(cache, q.requires_grad_(), table, lens)
    assert not calls
    with torch.no_grad():
        P.paged_attend(cache, q, table, lens)
    P.paged_attend(cache, q.detach(), table, lens)
    cache.k_pages = cache.k_pages.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        P.paged_attend(cache, q.detach(), table, lens)
    assert len(calls) == 2


def test_a_ring_that_is_left_early_waits_for_every_copy_in_flight():
    """The waits of a reader that gives up, on a model of the ring's barriers: for every ring, number of
    units and place to stop, each unit issued and not read is waited for, and its wait ends with its
    own copy and not before."""
    src = """
    #include <stdio.h>
    #include <vector>
    #include "paged.cuh"
    using namespace pbk::paged;
    int main() {
      long bad = 0, seen = 0;
      for (int stages = 1; stages <= 6; ++stages)
        for (int count = 0; count <= 40; ++count)
          for (int stop = 0; stop < count; ++stop) {
            std::vector<long> ended(stages, 0);  // phases of each stage's barrier that have ended
            auto open = [&](RingWait w) { return (ended[w.stage] & 1) == w.parity; };  // a wait would block
            long issued = count < stages ? count : stages;
            for (int u = 0; u < stop; ++u) {  // read, and the stage filled again
              if (!open(ring_wait(u, stages))) ++bad;
              ++ended[u % stages];
              if (open(ring_wait(u, stages))) ++bad;
              if (u + stages < count) ++issued;
            }
            if (ring_issued(stop, stages, count) != issued) ++bad;
            for (long u = stop; u < issued; ++u) {
              ++seen;
              if (!open(ring_wait(u, stages))) ++bad;  // would return with the copy in flight
            }
            for (long u = stop; u < issued; ++u) {
              ++ended[u % stages];
              if (open(ring_wait(u, stages))) ++bad;   // would wait for ever
            }
          }
      printf("%ld %ld", bad, seen);
    }
    """
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "ring.cpp"), os.path.join(d, "ring")
        with open(c, "w") as f:
            f.write(src)
        subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I",
                        os.path.join(ROOT, "pseudobrain_b200", "csrc"), "-I", "/usr/local/cuda/include", c, "-o", exe], check=True)
        bad, seen = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert bad == "0" and int(seen) > 10000


def test_append_takes_one_token_whose_key_and_value_rows_differ_in_stride(capi, monkeypatch):
    """Of a single token the stride between tokens means nothing: a key of its own beside a value
    inside a packed projection is taken; of two tokens it is refused."""
    import types

    import torch
    from pseudobrain_b200 import paged_cache as P
    calls = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(P, "LIB", types.SimpleNamespace(pbk_paged_append=lambda *a: calls.append(a) or 0))
    cache, _, table, lens = _host_cache(capi)
    packed = torch.zeros(2, 12, 64, dtype=torch.bfloat16)
    k, v = torch.zeros(2, 2, 64, dtype=torch.bfloat16), packed[:, 10:]
    P.paged_append_(cache, k[:1], v[:1], table[:1], lens[:1])
    assert calls[0][2:7] == (k.data_ptr(), v.data_ptr(), 128, 64, 1)
    with pytest.raises(ValueError, match="same strides"):
        P.paged_append_(cache, k, v, table[:2], lens[:2])
    assert len(calls) == 1
