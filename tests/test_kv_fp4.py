"""The 4-bit key/value cache on the CPU: what its entry points and the argument contract refuse, the scratch that an
attention asks for, the fake kernels, and which calls go to the custom ops."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from fused_decode import _lib as L
from fused_decode import kv_fp4, ops
from fused_decode._checks import check

E8M0 = torch.float8_e8m0fnu
# The entry points' checks return before any HIP call; no pointer is read.
nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
K, KS, V, VS, A, B, N, T, Y, P = (0x10000000 * i for i in range(1, 11))  # far apart


def refused(status, code, words):
    return status == code and words in L.lib().fd_last_error()


def shape(pages=6, heads=2, page=16, dim=64, step=None, head=None):
    head = page * dim // 2 if head is None else head
    return L.FdKvShape(pages, heads, page, dim, heads * head if step is None else step, head)


def append(k=K, ks=KS, v=V, vs=VS, s=None, a=A, b=B, st=(128, 128, 64, 128, 128, 64), n=N, t=T, ts=3, tp=3, seqs=2, new=1,
           act=0):
    return L.lib().fd_append_kv_fp4(k, ks, v, vs, s or shape(), a, b, *st, n, t, ts, tp, seqs, new, act, None)


def read(ok=A, ov=B, k=K, ks=KS, v=V, vs=VS, s=None, n=N, t=T, ts=3, tp=3, seqs=2, count=5, act=0):
    return L.lib().fd_read_kv_fp4(ok, ov, k, ks, v, vs, s or shape(), n, t, ts, tp, seqs, count, act, None)


def attend(y=Y, q=A, k=K, ks=KS, v=V, vs=VS, s=None, st=(256, 256, 64), n=N, t=T, ts=3, tp=3, seqs=2, new=1, hq=4,
           scale=0.1, scratch=None, size=0, act=0):
    return L.lib().fd_attend_kv_fp4(y, q, k, ks, v, vs, s or shape(), *st, n, t, ts, tp, seqs, new, hq, scale, scratch, size,
                                    act, None)


@nogpu
@pytest.mark.parametrize("call", [append, read, attend])
def test_the_entries_refuse(call):
    assert refused(call(act=2), L.FD_EINVAL, b"act_dtype")
    for name in ("k", "ks", "v", "vs", "n"):
        assert refused(call(**{name: None}), L.FD_EINVAL, b"null"), name
    for name in {append: ("a", "b"), read: ("ok", "ov"), attend: ("y", "q")}[call]:
        assert refused(call(**{name: None}), L.FD_EINVAL, b"null"), name
    for s in (shape(pages=-1), shape(heads=0), shape(page=0)):
        assert refused(call(s=s), L.FD_EINVAL, b"pages")
    for dim in (0, 32, 80, 100, 512):
        assert refused(call(s=shape(dim=dim)), L.FD_EUNSUPPORTED, b"dim")
    assert refused(call(s=shape(step=-16)), L.FD_EINVAL, b"negative")
    assert refused(call(s=shape(step=1032)), L.FD_EUNSUPPORTED, b"16 bytes")
    assert refused(call(s=shape(head=520, step=2048)), L.FD_EUNSUPPORTED, b"16 bytes")
    assert refused(call(s=shape(step=0)), L.FD_EINVAL, b"share") and refused(call(s=shape(head=496)), L.FD_EINVAL, b"share")
    assert refused(call(s=shape(pages=2**20, step=2**17)), L.FD_EUNSUPPORTED, b"GiB")
    assert refused(call(s=shape(pages=2**31)), L.FD_EUNSUPPORTED, b"large")
    assert refused(call(s=shape(heads=65536)), L.FD_EUNSUPPORTED, b"large")
    assert refused(call(seqs=65536), L.FD_EUNSUPPORTED, b"large")
    assert refused(call(k=K + 8), L.FD_EUNSUPPORTED, b"aligned") and refused(call(v=V + 1), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(call(t=None, seqs=7), L.FD_EINVAL, b"table")
    assert refused(call(ts=-1), L.FD_EINVAL, b"negative") and refused(call(tp=-1), L.FD_EINVAL, b"negative")
    assert refused(call(tp=2**28), L.FD_EUNSUPPORTED, b"tokens")
    assert refused(call(seqs=-1), L.FD_EINVAL, b"size")
    assert call(seqs=0) == L.FD_OK


@nogpu
def test_the_store_refuses():
    for i in range(6):
        st = [128, 128, 64, 128, 128, 64]
        st[i] = -1
        assert refused(append(st=st), L.FD_EINVAL, b"stride")
    assert append(new=0) == L.FD_OK and append(tp=0) == L.FD_OK and refused(append(new=-1), L.FD_EINVAL, b"size")
    codes, scales = 6 * 2 * 16 * 32, 6 * 2 * 16 * 2
    for name, at, size in (("v", K, codes), ("vs", KS, scales), ("ks", K, codes), ("vs", V, codes), ("v", KS - codes, codes)):
        assert refused(append(**{name: at + size - 16}), L.FD_EINVAL, b"each other"), name
    new = 2 * 128 * 2  # bytes
    for at, size in ((K, codes), (KS, scales), (V, codes), (VS, scales)):
        for name in ("a", "b"):
            for where in (at, at + size - 1, at - new + 1):
                assert refused(append(**{name: where}), L.FD_EINVAL, b"stored"), name
        assert refused(append(n=at + size - 1), L.FD_EINVAL, b"stored")
        assert refused(append(t=at - 23), L.FD_EINVAL, b"stored")


@nogpu
def test_the_read_refuses():
    assert read(count=0) == L.FD_OK and refused(read(count=-1), L.FD_EINVAL, b"size")
    assert refused(read(ok=A + 8), L.FD_EUNSUPPORTED, b"aligned")
    n = 2 * 5 * 2 * 64 * 2
    assert refused(read(ov=A + n - 16), L.FD_EINVAL, b"each other")
    for at in (K, KS, V, VS, N, T):
        assert refused(read(ok=at), L.FD_EINVAL, b"overlap") and refused(read(ov=at - n + 16), L.FD_EINVAL, b"overlap")
    assert refused(read(count=2**31 - 1), L.FD_EUNSUPPORTED, b"large")


@nogpu
def test_the_attention_refuses():
    for st in ((-1, 256, 64), (256, -1, 64), (256, 256, -1)):
        assert refused(attend(st=st), L.FD_EINVAL, b"stride")
    assert refused(attend(hq=3), L.FD_EINVAL, b"multiple")
    assert attend(new=0) == L.FD_OK and attend(hq=0) == L.FD_OK
    for scale in (float("nan"), float("inf"), 3e38):
        assert refused(attend(scale=scale), L.FD_EINVAL, b"scale")
    assert refused(attend(y=Y + 2), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(attend(scratch=P + 8, size=100), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(attend(s=shape(pages=0)), L.FD_EUNSUPPORTED, b"without pages")
    n = 2 * 4 * 64 * 2
    for at in (A, K, KS, V, VS, N, T):
        assert refused(attend(y=at), L.FD_EUNSUPPORTED, b"overlap") and refused(attend(y=at - n + 16), L.FD_EUNSUPPORTED,
                                                                                b"overlap")
    assert refused(attend(new=600000, y=Y << 8), L.FD_EUNSUPPORTED, b"rows")


def test_scratch_sizes():
    def size(b, n, hq, heads, dim, capacity):
        out = ctypes.c_int64(-1)
        return L.lib().fd_attend_kv_fp4_scratch(b, n, hq, heads, dim, capacity, ctypes.byref(out)), out.value

    assert size(-1, 1, 4, 2, 64, 10)[0] == L.FD_EINVAL and size(1, 1, 3, 2, 64, 10)[0] == L.FD_EINVAL
    assert size(1, 1, 4, 0, 64, 10)[0] == L.FD_EINVAL and size(1, 1, 4, 2, 80, 10)[0] == L.FD_EUNSUPPORTED
    assert L.lib().fd_attend_kv_fp4_scratch(1, 1, 4, 2, 64, 10, None) == L.FD_EINVAL
    for b, n, hq in ((0, 1, 4), (1, 0, 4), (1, 1, 0)):
        assert size(b, n, hq, 2, 64, 100000) == (L.FD_OK, 0)
    assert size(1, 1, 4, 2, 64, 100) == (L.FD_OK, 0)  # one share
    status, some = size(1, 1, 32, 8, 128, 131072)
    assert status == L.FD_OK and some > 0 and some % (8 * 16 * 132 * 4) == 0


# ------------------------------------------------------------------ the contract and where a call goes


def cuda(*size, dtype=torch.float16):
    return torch.empty(size, dtype=dtype, device="cuda")


def fake_cache(pages=6, heads=2, page=16, dim=64):
    c = lambda: cuda(pages, heads, page, dim // 2, dtype=torch.uint8)
    s = lambda: cuda(pages, heads, page, dim // 32, dtype=E8M0)
    return dict(k=c(), k_scale=s(), v=c(), v_scale=s())


def test_the_contract_of_a_cache():
    with FakeTensorMode():
        n = cuda(2, dtype=torch.int32)
        given = lambda **other: check("read_kv_fp4", **{**dict(**fake_cache(), lengths=n, count=3, pages=None,
                                                              dtype=torch.float16), **other})
        given()
        # a layer of a tensor of several, and every second page
        layers = {name: torch.empty(6, 5, *t.shape[1:], dtype=t.dtype, device="cuda")[:, 2]
                  for name, t in fake_cache().items()}
        given(**layers), given(**{name: t[::2] for name, t in fake_cache().items()})
        given(pages=cuda(2, 3, dtype=torch.int32), count=0)
        for wrong in (dict(k=None), dict(k=cuda(6, 2, 16, 32)), dict(v_scale=cuda(6, 2, 16, 2, dtype=torch.uint8)),
                      dict(lengths=[1]), dict(lengths=cuda(2, dtype=torch.int64)), dict(pages=3), dict(count=2.5),
                      dict(pages=cuda(2, 3)), dict(count=None), dict(count=True), dict(dtype=torch.float32)):
            with pytest.raises(TypeError):
                given(**wrong)
        big = fake_cache(page=32)
        for wrong in (dict(k=cuda(6, 2, 16, 16, dtype=torch.uint8)), dict(v=cuda(6, 2, 8, 32, dtype=torch.uint8)),
                      dict(k_scale=cuda(6, 2, 16, 1, dtype=E8M0)), dict(k=cuda(2, 16, 32, dtype=torch.uint8)),
                      dict(v=cuda(6, 2, 32, 32, dtype=torch.uint8)[:, :, ::2]), dict(v=big["v"][:, :, :16]),
                      dict(k=cuda(6, 16, 2, 32, dtype=torch.uint8).transpose(1, 2)), dict(count=-1),
                      dict(lengths=cuda(1, 2, dtype=torch.int32)), dict(lengths=cuda(7, dtype=torch.int32)),
                      dict(pages=cuda(3, 3, dtype=torch.int32)), dict(pages=cuda(2, dtype=torch.int32)),
                      fake_cache(heads=0), fake_cache(page=0), fake_cache(dim=160)):
            with pytest.raises(ValueError):
                given(**wrong)


def test_the_contract_of_stores_and_queries():
    with FakeTensorMode():
        n, new = cuda(2, dtype=torch.int32), cuda(2, 3, 2, 64)
        store = lambda **other: check("append_kv_fp4", **{**dict(**fake_cache(), new_k=new, new_v=new, lengths=n, pages=None),
                                                          **other})
        query = lambda **other: check("attend_kv_fp4", **{**dict(**fake_cache(), q=cuda(2, 3, 8, 64), lengths=n, pages=None,
                                                                 scale=None, out=None), **other})
        store()
        assert query()["scale"] == 0.125 and query(scale=2)["scale"] == 2.0
        query(out=cuda(2, 3, 8, 64))
        for wrong in (dict(new_k=None), dict(new_k=cuda(2, 3, 2, 64, dtype=torch.float32)),
                      dict(new_v=cuda(2, 3, 2, 64, dtype=torch.bfloat16)), dict(new_v=1)):
            with pytest.raises(TypeError):
                store(**wrong)
        for wrong in (dict(new_k=cuda(2, 3, 4, 64)), dict(new_k=cuda(2, 3, 2, 32)), dict(new_k=cuda(3, 2, 64)),
                      dict(new_v=cuda(2, 2, 2, 64)), dict(new_k=cuda(1, 3, 2, 64), new_v=cuda(1, 3, 2, 64))):
            with pytest.raises(ValueError):
                store(**wrong)
        for wrong in (dict(q=cuda(2, 3, 8, 64, dtype=torch.float32)), dict(q=None), dict(out=3),
                      dict(out=cuda(2, 3, 8, 64, dtype=torch.bfloat16))):
            with pytest.raises(TypeError):
                query(**wrong)
        for wrong in (dict(q=cuda(2, 3, 7, 64)), dict(q=cuda(2, 3, 8, 128)), dict(q=cuda(2, 8, 64)), dict(scale="a"),
                      dict(scale=float("inf")), dict(scale=2e38), dict(q=cuda(1, 3, 8, 64)),
                      dict(out=cuda(2, 8, 3, 64).transpose(1, 2)), dict(out=cuda(2, 3, 8, 32))):
            with pytest.raises(ValueError):
                query(**wrong)


def cpu_cache(pages=6, heads=2, page=16, dim=64):
    return kv_fp4.KvCacheFp4.empty(pages, heads, page, dim, device="cpu")


def test_tensors_off_the_gpu_and_wrong_caches_are_refused():
    c, n = cpu_cache(), torch.tensor([3, 4], dtype=torch.int32)
    new, q = torch.zeros(2, 1, 2, 64).half(), torch.zeros(2, 1, 4, 64).half()
    f = torch.ops.fused_decode
    for call in (lambda: kv_fp4.append_kv_fp4(c, new, new, n), lambda: kv_fp4.read_kv_fp4(c, n, 3),
                 lambda: kv_fp4.attend_kv_fp4(q, c, n), lambda: f.append_kv_fp4(*c, new, new, n),
                 lambda: f.read_kv_fp4(*c, n, 3), lambda: f.attend_kv_fp4(q, *c, n)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for wrong in (None, c[:3], 7, torch.zeros(4), [1, 2, 3, 4]):
        for call in (lambda: kv_fp4.append_kv_fp4(wrong, new, new, n), lambda: kv_fp4.read_kv_fp4(wrong, n, 3),
                     lambda: kv_fp4.attend_kv_fp4(q, wrong, n)):
            with pytest.raises((TypeError, ValueError)):
                call()
    for call in (lambda: kv_fp4.append_kv_fp4(c, None, new, n), lambda: kv_fp4.read_kv_fp4(c, None, 3),
                 lambda: kv_fp4.attend_kv_fp4(None, c, n), lambda: kv_fp4.attend_kv_fp4(q, c, n, 5)):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_the_fake_kernels_and_a_traced_graph():
    with FakeTensorMode():
        c = kv_fp4.KvCacheFp4(*fake_cache().values())
        n, new, q = cuda(2, dtype=torch.int32), cuda(2, 3, 2, 64), cuda(2, 8, 3, 64).transpose(1, 2)
        assert kv_fp4.append_kv_fp4(c, new, new, n) is None
        k, v = kv_fp4.read_kv_fp4(c, n, 9)
        assert k.shape == v.shape == (2, 9, 2, 64) and k.dtype == torch.bfloat16
        y = kv_fp4.attend_kv_fp4(q, c, n)
        assert y.shape == q.shape and y.is_contiguous() and y.dtype == torch.float16

        def f(k, ks, v, vs, new, n, q):
            c = kv_fp4.KvCacheFp4(k, ks, v, vs)
            kv_fp4.append_kv_fp4(c, new, new, n)
            return kv_fp4.attend_kv_fp4(q, c, n)

        graph = make_fx(f)(*c, new, n, q).graph
    names = [str(node.target) for node in graph.nodes if node.op == "call_function"]
    assert sum("append_kv_fp4" in t for t in names) == 1 and sum("attend_kv_fp4" in t for t in names) == 1


class Calls(list):
    """Stands in for the native binding: notes each call and returns FD_OK."""

    def __getattr__(self, name):
        def call(*args):
            self.append((name, args))
            return L.FD_OK
        return call


@pytest.fixture
def calls(monkeypatch):
    stand_in = Calls()
    monkeypatch.setattr(kv_fp4, "native", lambda: stand_in)
    monkeypatch.setattr(kv_fp4, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(kv_fp4, "_current_device", lambda: None)  # the CPU's index
    monkeypatch.setattr(kv_fp4._lib, "scratch_bytes", lambda *a: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(kv_fp4, "check", lambda op, **a: a)
    ops.clear_plans()
    yield stand_in
    ops.clear_plans()


def test_calls_launch_once_and_keep_a_plan(calls):
    c, n = cpu_cache(), torch.tensor([3, 4], dtype=torch.int32)
    new, q = torch.zeros(2, 1, 2, 64).half(), torch.zeros(2, 1, 4, 64).half()
    before = [t._version for t in c]
    for _ in range(2):
        kv_fp4.append_kv_fp4(c, new, new, n)
        kv_fp4.read_kv_fp4(c, n, 3)
        kv_fp4.attend_kv_fp4(q, c, n, scale=0.5)
    assert [name for name, _ in calls] == ["append_kv_fp4", "read_kv_fp4", "attend_kv_fp4"] * 2 and len(ops._PLANS) == 3
    assert all(t._version > b for t, b in zip(c, before))
    for name, args in calls:  # every call gets the struct of its plan, alive
        at = args[{"append_kv_fp4": 4, "read_kv_fp4": 6, "attend_kv_fp4": 6}[name]]
        s = L.FdKvShape.from_address(at)
        assert (s.pages, s.heads, s.page, s.dim, s.page_stride, s.head_stride) == (6, 2, 16, 64, 1024, 512)
    out = torch.empty(2, 1, 4, 64).half()
    assert kv_fp4.attend_kv_fp4(q, c, n, scale=0.5, out=out) is out and out._version > 0
    # what is not dense along its rows goes as a copy
    spread = torch.zeros(2, 1, 2, 128).half()[..., ::2]
    kv_fp4.append_kv_fp4(c, spread, new, n)
    args = calls[-1][1]
    assert args[5] != spread.data_ptr() and args[6] == new.data_ptr() and args[7:10] == (128, 128, 64)
    table = torch.zeros(3, 2, dtype=torch.int32).t()
    kv_fp4.read_kv_fp4(c, torch.zeros(4, dtype=torch.int32)[::2], 3, table)
    args = calls[-1][1]
    assert args[8] != table.data_ptr() and args[9:11] == (3, 3)
    one = torch.zeros(2, 9, dtype=torch.int32)[:, 2:5]
    kv_fp4.read_kv_fp4(c, n, 3, one)
    assert calls[-1][1][8] == one.data_ptr() and calls[-1][1][9:11] == (9, 3)


def test_a_cache_of_no_pages_shows_zeros(calls):
    c, n = cpu_cache(pages=0), torch.tensor([3], dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    out = torch.ones(1, 1, 4, 64).half()
    assert not kv_fp4.attend_kv_fp4(out, c, n, table, scale=1.0).any() and calls == []
    q = out.clone()
    assert kv_fp4.attend_kv_fp4(q, c, n, table, scale=1.0, out=out) is out and not out.any()


def test_recorded_calls_go_to_the_custom_ops(calls, monkeypatch):
    c, n = cpu_cache(), torch.tensor([3, 4], dtype=torch.int32)
    new, q = torch.zeros(2, 1, 2, 64).half(), torch.zeros(2, 1, 4, 64).half()
    seen = []

    class Stand:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or torch.zeros(2, 1, 4, 64).half()

    monkeypatch.setattr(torch.ops, "fused_decode", Stand(), raising=False)
    leaf, neg = lambda t: t.clone().requires_grad_(), torch._neg_view
    kv_fp4.append_kv_fp4(c, leaf(new), new, n), kv_fp4.append_kv_fp4(c, new, neg(new), n)
    kv_fp4.attend_kv_fp4(leaf(q), c, n), kv_fp4.attend_kv_fp4(neg(q), c, n)
    assert calls == [] and seen == ["append_kv_fp4"] * 2 + ["attend_kv_fp4"] * 2
    with torch.no_grad():
        kv_fp4.attend_kv_fp4(leaf(q), c, n, scale=1.0)
    assert len(calls) == 1
