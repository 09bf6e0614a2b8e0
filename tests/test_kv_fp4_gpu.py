"""The 4-bit key/value cache: stores bit for bit against ``quantize_fp4`` on the CPU, reads against the values that codes
stand for, and attention against float64.

Attention. A score's float32 evaluation (2 D products of exact numbers and their sum, a float16 query's two parts, the
scale) is off by e = (2.1 D + 8) * 2^-23 of scale * sum |q k|; so is p = exp(score - max) relative, twice with the
maximum's own error, plus 2^-21 of the largest |score| for the exponent's rounding and the exponential's, and 2^-16 for
its two bfloat16 parts. A sum of n tokens, rescaled at most once a step of 32, adds (n + 64) * 2^-23. So y is off by at
most twice (numerator and denominator) all of these times sum p |v| / sum p, before half a step of its type."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float16: (2.0**-11, 2.0**-25), torch.bfloat16: (2.0**-8, 2.0**-134)}
BOTH = [torch.float16, torch.bfloat16]
DIMS = [64, 96, 128, 192, 256]
E8M0 = torch.float8_e8m0fnu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed)) * scale).to(dtype).to(DEV)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def random_cache(pages, heads, page, dim, seed, lo=-3, hi=0):
    """Any codes, scales of 2^lo .. 2^hi."""
    import fused_decode as fd

    t = []
    for i in range(2):
        t.append(torch.randint(0, 256, (pages, heads, page, dim // 2), generator=gen(seed + i), dtype=torch.uint8).to(DEV))
        s = torch.randint(127 + lo, 128 + hi, (pages, heads, page, dim // 32), generator=gen(seed + 2 + i), dtype=torch.uint8)
        t.append(s.to(DEV).view(E8M0))
    return fd.KvCacheFp4(*t)


def values64(codes, scale):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long().cpu()
    s = scale.view(torch.uint8).cpu().double()
    s = torch.where(s == 255, float("nan"), torch.exp2(s - 127)).repeat_interleave(32, -1)
    return GRID[c & 7] * (1 - 2 * (c >> 3)) * s


def tokens64(cache, b, table, length):
    """What sequence b's tokens hold, keys and values [heads, n, dim], and whether each is in the cache, on the CPU."""
    pages, heads, page, half = cache.k.shape
    capacity = page if table is None else table.shape[1] * page
    n = max(0, min(int(length), capacity))
    rows = [b] * (n // page + 1) if table is None else table[b].tolist()
    at = [(rows[t // page], t % page) for t in range(n)]
    here = torch.tensor([0 <= r < pages for r, _ in at], dtype=torch.bool)
    out = []
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        v = values64(codes, scale)
        out.append(torch.stack([v[r, :, s] if 0 <= r < pages else torch.zeros(heads, 2 * half).double() for r, s in at], 1)
                   if n else torch.zeros(heads, 0, 2 * half).double())
    return (*out, here)


def check_attention(y, q, cache, lengths, table=None, scale=None):
    b_, new, hq, dim = q.shape
    heads = cache.k.shape[1]
    group = hq // heads
    scale = dim**-0.5 if scale is None else scale
    half, least = HALF_STEP[q.dtype]
    got = y.cpu().double()
    assert y.shape == q.shape and y.dtype == q.dtype and y.is_contiguous()
    for b in range(b_):
        length = int(lengths[b])
        k, v, here = tokens64(cache, b, table, length)
        for i in range(new):
            to = length - new + i + 1
            n = max(0, min(to, k.shape[1]))
            mask = here[:n]
            if not bool(mask.any()):
                assert not got[b, i].any(), (b, i)
                continue
            qq = q[b, i].cpu().double().view(heads, group, dim)
            kk, vv = k[:, :n][:, mask], v[:, :n][:, mask]
            s = qq @ kk.transpose(1, 2) * scale
            p = torch.softmax(s, -1)
            want, mag = p @ vv, p @ vv.abs()
            e = (2.1 * dim + 8) * 2.0**-23 * abs(scale) * (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1)
            rel = 2 * e + 2.0**-21 * s.abs().amax(-1) + 2.0**-16 + (n + 64) * 2.0**-23
            err = 2 * rel[..., None] * mag
            g = got[b, i].view(heads, group, dim)
            ok = (g - want).abs() <= err + half * (want.abs() + err) + least
            assert bool(ok.all()), (b, i, length, float((g - want).abs().max()))


CASES = [  # sequences, new, heads, group, page (0: no table), lengths
    (1, 1, 1, 1, 0, [1]), (2, 1, 2, 4, 0, [31, 32]), (3, 1, 2, 3, 16, [33, 64, 129]), (2, 2, 1, 5, 24, [2, 100]),
    (2, 5, 3, 4, 7, [60, 5]), (1, 17, 2, 1, 64, [200]), (1, 3, 1, 16, 32, [77]), (2, 1, 1, 17, 100, [300, 1]),
    (4, 1, 2, 2, 1, [5, 40, 0, 3]), (2, 1, 4, 8, 256, [700, 512]), (1, 16, 1, 8, 48, [333])]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("b,new,heads,group,page,lengths", CASES)
def test_attention(b, new, heads, group, page, lengths, dim, dtype):
    import fused_decode as fd

    most = max(lengths)
    if page:
        per = -(-most // page)
        cache = random_cache(b * per + 3, heads, page, dim, seed=dim)
        table = torch.randperm(b * per + 3, generator=gen(b))[: b * per].view(b, per).to(torch.int32).to(DEV)
    else:
        cache, table = random_cache(b, heads, most + 5, dim, seed=dim), None
    q = rnd(b, new, heads * group, dim, seed=1, dtype=dtype)
    n = i32(lengths)
    check_attention(fd.attend_kv_fp4(q, cache, n, table), q, cache, n, table)
    y = fd.attend_kv_fp4(q, cache, n, table, scale=-0.3)
    check_attention(y, q, cache, n, table, -0.3)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim,page,length", [(128, 64, 20000), (64, 128, 5000), (256, 0, 3000), (96, 40, 9999), (192, 16, 4112)])
def test_attention_over_many_shares(dim, page, length, dtype):
    """Long sequences next to short ones: tokens cut into shares, some of them empty, and joined."""
    import fused_decode as fd

    size = page or length + 11
    lengths = [length, 1, 0, 200]
    per = -(-length // size)
    cache = random_cache(len(lengths) * per, 2, size, dim, seed=1)
    table = torch.randperm(len(lengths) * per, generator=gen(3)).view(4, per).to(torch.int32).to(DEV) if page else None
    q = rnd(4, 2, 6, dim, seed=2, dtype=dtype, scale=2.0)
    n = i32(lengths)
    check_attention(fd.attend_kv_fp4(q, cache, n, table), q, cache, n, table)


@pytest.mark.parametrize("dim", DIMS)
def test_lengths_and_pages_outside_the_cache(dim):
    """Tokens past the pages, lengths below zero, page numbers that no page has: neither read nor seen."""
    import fused_decode as fd

    cache = random_cache(9, 2, 16, dim, seed=1)
    table = i32([[0, 3, 8], [9, 1, -1], [-5, 1 << 30, 2], [4, 4, 4], [-1, -1, 9], [5, 6, 7]])
    q = rnd(6, 3, 4, dim, seed=2, dtype=torch.bfloat16)
    for lengths in ([48, 40, 44, 47, 30, 33], [49, 1000, 2**31 - 1, 2, -3, -(2**31)], [50, 17, 16, 15, 0, 51]):
        n = i32(lengths)
        check_attention(fd.attend_kv_fp4(q, cache, n, table), q, cache, n, table)
        k, v = fd.read_kv_fp4(cache, n, 60, table, dtype=torch.float16)
        for b in range(6):
            kk, vv, here = tokens64(cache, b, table, lengths[b])
            for got, want in ((k, kk), (v, vv)):
                m = want.shape[1]
                want = torch.where(here[None, :, None], want, 0.0).transpose(0, 1)
                assert torch.equal(got[b, :m].cpu().double(), want) and not got[b, m:].any()
    before = [t.clone() for t in cache]
    fd.append_kv_fp4(cache, rnd(6, 3, 2, dim, seed=3, dtype=torch.float16), rnd(6, 3, 2, dim, seed=4, dtype=torch.float16),
                     i32([49, 35, 20, 2, 3, -4]), table)
    kept = torch.ones(9, 16, dtype=torch.bool)
    for page, slots in ((8, (14, 15)), (4, (0, 1))):  # of 46 .. 48 two lie in pages; 32 .. 34 and 17 .. 19 in none; 0, 1
        kept[page, list(slots)] = False
    for t, old in zip(cache, before):
        same = (t.view(torch.uint8) == old.view(torch.uint8)).all(-1).cpu()
        assert bool(same.transpose(1, 2)[kept].all()) and not bool(same.transpose(1, 2)[~kept].all())


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("dtype", BOTH)
def test_what_is_not_a_number_stays_with_those_who_see_it(dim, dtype):
    """NaN scales: in slots behind a sequence's end nobody's, of one token's values only its later queries' and its own
    group's, of its keys every later query's."""
    import fused_decode as fd

    cache = random_cache(2, 2, 80, dim, seed=1)
    q, n = rnd(2, 6, 4, dim, seed=2, dtype=dtype), i32([50, 64])
    for scale in (cache.k_scale, cache.v_scale):
        raw = scale.view(torch.uint8)
        raw[0, :, 50:], raw[1, :, 64:] = 255, 255
    y = fd.attend_kv_fp4(q, cache, n)
    clean = fd.KvCacheFp4(cache.k, cache.k_scale.view(torch.uint8).clamp(max=127).view(E8M0), cache.v,
                          cache.v_scale.view(torch.uint8).clamp(max=127).view(E8M0))
    assert torch.equal(y, fd.attend_kv_fp4(q, clean, n))
    raw = cache.v_scale.view(torch.uint8)
    held = raw[0, 1, 47, 1].item()
    raw[0, 1, 47, 1] = 255  # token 47: seen by queries 3 .. 5 of tokens 45 .. 50
    got = fd.attend_kv_fp4(q, cache, n)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 3 - 1 :, 2:, 32:64] = True  # queries are tokens 44 .. 49
    bad[0, 2, 2:] = False
    assert bool(torch.isnan(got[bad]).all()) and not bool(torch.isnan(got[~bad]).any())
    check_attention(got[:, :3].contiguous(), q[:, :3], clean, n - 3)
    raw[0, 1, 47, 1] = held
    cache.k_scale.view(torch.uint8)[1, 0, 62, 0] = 255
    got = fd.attend_kv_fp4(q, cache, n)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, 4:, :2] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], y[~bad])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
def test_stores_are_the_quantisers(dim, dtype):
    """Every slot of the tokens has quantize_fp4's codes and scales, every other slot what it had."""
    import fused_decode as fd

    for new, page, heads, lengths in ((1, 16, 1, [1, 16, 17]), (5, 7, 3, [5, 3, 30]), (40, 24, 2, [40, 47, 100])):
        per = -(-max(lengths) // page)
        cache = random_cache(3 * per + 1, heads, page, dim, seed=5)
        table = torch.randperm(3 * per + 1, generator=gen(new))[: 3 * per].view(3, per).to(torch.int32).to(DEV)
        k = rnd(3, new, heads, dim, seed=6, dtype=dtype) * torch.exp2(rnd(3, new, 1, 1, seed=7, scale=4.0)).to(dtype)
        v = rnd(3, new, heads, dim, seed=8, dtype=dtype)
        v[0, 0, 0, :32] = 0.0
        v[1, -1, 0, 3], k[2, 0, 0, 33] = float("inf"), float("nan")
        k[0, 0, 0, :32] = torch.finfo(dtype).smallest_normal / 2
        want = [t.cpu().view(torch.uint8).clone() for t in cache]
        for src, at in ((k, 0), (v, 2)):
            codes, scale = fd.quantize_fp4(src.cpu().reshape(-1, dim))
            codes, scale = codes.view(3, new, heads, -1), scale.view(torch.uint8).view(3, new, heads, -1)
            for b, length in enumerate(lengths):
                for i in range(new):
                    t = length - new + i
                    if t >= 0:
                        want[at][int(table[b, t // page]), :, t % page] = codes[b, i]
                        want[at + 1][int(table[b, t // page]), :, t % page] = scale[b, i]
        fd.append_kv_fp4(cache, k, v, i32(lengths), table)
        for t, w in zip(cache, want):
            assert torch.equal(t.view(torch.uint8).cpu(), w)


@pytest.mark.parametrize("dim", DIMS)
def test_reads(dim):
    import fused_decode as fd

    cache = random_cache(8, 3, 10, dim, seed=1, lo=-20, hi=20)
    cache.v_scale.view(torch.uint8)[3, 1, 4, 0] = 255
    for table, lengths, count in ((i32([[3, 1], [0, 7]]), [20, 13], 20), (i32([[3, 1], [0, 7]]), [4, 7], 5),
                                  (None, [10, 9, 8, 7, 6, 5, 0], 13), (None, [3], 1), (i32([[3, 2, 1]])[:, :0], [9], 4)):
        for dtype in BOTH:
            got = fd.read_kv_fp4(cache, i32(lengths), count, table, dtype=dtype)
            for b, length in enumerate(lengths):
                for g, want in zip(got, tokens64(cache, b, table, min(length, count))[:2]):
                    assert g.shape == (len(lengths), count, 3, dim) and g.dtype == dtype
                    m = want.shape[1]
                    want = want.transpose(0, 1).to(dtype)
                    assert torch.equal(torch.nan_to_num(g[b, :m].cpu(), 1e4), torch.nan_to_num(want, 1e4))
                    assert not g[b, m:].any()
    assert fd.read_kv_fp4(cache, i32([1]), 0)[0].shape == (1, 0, 3, dim)
    assert fd.read_kv_fp4(cache, i32([]), 3)[0].shape == (0, 3, 3, dim)


@pytest.mark.parametrize("dtype", BOTH)
def test_views_of_every_operand(dtype):
    """A cache that is one layer of several, queries and new tokens of one projection's output, tables and lengths with
    strides of their own, outputs given."""
    import fused_decode as fd

    dim, heads, group, page = 128, 2, 4, 16
    whole = random_cache(12, 3 * heads, page, dim, seed=1)
    layer = fd.KvCacheFp4(*(t.view(12, 3, heads, *t.shape[2:])[::2, 1] for t in whole))
    dense = fd.KvCacheFp4(*(t.view(torch.uint8).clone().view(t.dtype) for t in layer))
    before = [t.view(torch.uint8).clone() for t in whole]
    qkv = rnd(3, 1, heads * (group + 2), dim, seed=2, dtype=dtype)
    q, k, v = qkv.split([heads * group, heads, heads], dim=2)
    table = i32([[0, 1, 9], [2, 3, 9], [4, 5, 9]]).t().contiguous().t()[:, :2]
    lengths = i32([[20, 0], [32, 0], [1, 0]])[:, 0]
    for c in (layer, dense):
        fd.append_kv_fp4(c, k, v, lengths, table)
    for a, b in zip(layer, dense):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for t, old in zip(whole, before):  # other layers and pages
        t = t.view(torch.uint8).view(12, 3, heads, *t.shape[2:])
        old = old.view(t.shape)
        assert torch.equal(t[1::2], old[1::2]) and torch.equal(t[:, ::2], old[:, ::2])
    y = fd.attend_kv_fp4(q, layer, lengths, table)
    check_attention(y, q, dense, lengths, table)
    out = torch.empty_like(y)
    assert fd.attend_kv_fp4(q, layer, lengths, table, out=out) is out and torch.equal(out, y)
    odd = torch.empty(y.numel() + 1, dtype=dtype, device=DEV)[1:].view(y.shape)  # off 16-byte alignment
    assert fd.attend_kv_fp4(q, layer, lengths, table, out=odd) is odd and torch.equal(odd, y)
    own = q.contiguous()
    assert fd.attend_kv_fp4(own, layer, lengths, table, out=own) is own and torch.equal(own, y)
    spread = torch.zeros(3, 1, heads * group, 2 * dim, dtype=dtype, device=DEV)[..., ::2]
    spread.copy_(q)
    assert torch.equal(fd.attend_kv_fp4(spread, layer, lengths, table), y)
    shared = rnd(1, 1, heads * group, dim, seed=3, dtype=dtype).expand(3, -1, -1, -1)
    check_attention(fd.attend_kv_fp4(shared, layer, lengths, table), shared, dense, lengths, table)
    for a, b in zip(fd.read_kv_fp4(layer, lengths, 32, table, dtype=dtype), fd.read_kv_fp4(dense, lengths, 32, table, dtype=dtype)):
        assert torch.equal(a, b)
    empty = q[:0]
    assert fd.attend_kv_fp4(empty, layer, lengths[:0], table[:0]).shape == empty.shape
    fd.append_kv_fp4(layer, k[:0], v[:0], lengths[:0], table[:0])
    assert fd.attend_kv_fp4(q, layer, lengths, table[:, :0]).count_nonzero() == 0


def test_large_scores():
    """Scores of some thousands, all but one weight 0, and equal ones."""
    import fused_decode as fd

    cache = random_cache(1, 1, 300, 128, seed=1, lo=2, hi=4)
    q = rnd(1, 1, 3, 128, seed=2, dtype=torch.bfloat16, scale=8.0)
    check_attention(fd.attend_kv_fp4(q, cache, i32([300]), scale=1.0), q, cache, i32([300]), scale=1.0)
    cache.k.fill_(0x22)
    cache.k_scale.view(torch.uint8).fill_(127)
    y = fd.attend_kv_fp4(q, cache, i32([300]))
    check_attention(y, q, cache, i32([300]))


def test_a_step_captured_and_replayed():
    """Store and attention in a graph whose lengths and pages change between replays, two graphs of one signature in
    turn, and the eager calls between them."""
    import fused_decode as fd

    caches = [random_cache(40, 2, 16, 128, seed=s) for s in (1, 2)]
    mirror = [fd.KvCacheFp4(*(t.view(torch.uint8).clone().view(t.dtype) for t in c)) for c in caches]
    q, k, v = (rnd(4, 1, h, 128, seed=s, dtype=torch.float16) for h, s in ((8, 3), (2, 4), (2, 5)))
    lengths, table = i32([30, 100, 1, 160]), torch.randperm(40, generator=gen(1)).view(4, 10).to(torch.int32).to(DEV)

    def step(c):
        fd.append_kv_fp4(c, k, v, lengths, table)
        return fd.attend_kv_fp4(q, c, lengths, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, step(mirror[0]))
    graphs = []
    for c in caches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step(c)
        graphs.append((graph, y))
    for i in range(1, 5):
        lengths.copy_(i32([30 + i, 100 + 15 * i, i, 160 - 20 * i]))
        table.copy_(table.roll(1, 1))
        for t, s in ((q, 10), (k, 20), (v, 30)):
            t.copy_(rnd(*t.shape, seed=s + i, dtype=torch.float16))
        for (graph, y), c, m in zip(graphs, caches, mirror):
            graph.replay()
            want = step(m)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, m))


@pytest.mark.parametrize("dtype", BOTH)
def test_a_layer_held_in_four_bits(dtype):
    """Norm, QKV, rotation, store, attention, output projection, the norms around the block and the MLP, for two tokens
    in turn, against the same layer composed of the framework's 16-bit operators and torch on the dequantised weights."""
    import fused_decode as fd

    h, i, heads, kv, dim, b = 512, 768, 4, 2, 128, 3
    g = lambda *s, seed, scale=1.0, mean=0.0: rnd(*s, seed=seed, scale=scale) + mean
    w = {name: fd.quantize_fp4(g(n, k, seed=s, scale=k**-0.5)) for s, (name, n, k) in enumerate(
        (("qkv", (heads + 2 * kv) * dim, h), ("o", h, heads * dim), ("gu", 2 * i, h), ("down", h, i)))}
    norms = [g(h, seed=20 + j, scale=0.1, mean=1.0).to(dtype) for j in range(4)]
    cache = fd.KvCacheFp4.empty(6, kv, 16, dim)
    table, base = i32([[0, 1], [2, 3], [4, 5]]), i32([0, 3, 15])
    fd.append_kv_fp4(cache, *(rnd(3, 15, kv, dim, seed=s, dtype=dtype) for s in (30, 31)), base, table)
    dq = {name: fd.dequantize_fp4(*c).to(torch.float32) for name, c in w.items()}
    for t in range(2):
        x = rnd(b, h, seed=40 + t, dtype=dtype)
        lengths = base + t + 1
        ang = torch.outer(lengths.float() - 1, 10000.0 ** (-torch.arange(0, dim, 2, device=DEV) / dim))
        cos, sin = (f(torch.cat([ang, ang], -1)).view(b, 1, dim) for f in (torch.cos, torch.sin))
        normed = fd.rms_norm(x, norms[0], 1e-5)
        qkv = fd.linear_fp4(normed, *w["qkv"]).view(b, heads + 2 * kv, dim)
        qk = fd.rope(qkv[:, : heads + kv], cos, sin).unsqueeze(1)
        fd.append_kv_fp4(cache, qk[:, :, heads:], qkv[:, heads + kv :].unsqueeze(1), lengths, table)
        att = fd.attend_kv_fp4(qk[:, :, :heads], cache, lengths, table)
        out = fd.linear_fp4(att.view(b, -1), *w["o"])
        y, stream = fd.norm_add_norm(out, x, norms[1], norms[2], 1e-5)
        mid = fd.linear_fp4(y, *w["gu"], activation="swiglu")
        last, stream2 = fd.norm_add_norm(fd.linear_fp4(mid, *w["down"]), stream, norms[3], norms[0], 1e-5)
        # each step against its parts: the projections against float32 products of the decoded weights
        tol = dict(rtol=2.0 ** (-7 if dtype is torch.bfloat16 else -10), atol=2.0 ** (-8 if dtype is torch.bfloat16 else -11))
        close = lambda a, b: torch.testing.assert_close(a.float(), b.float(), **tol)
        close(qkv.flatten(1), (normed.float() @ dq["qkv"].t()).to(dtype))
        check_attention(att, qk[:, :, :heads], cache, lengths, table)
        close(out, (att.view(b, -1).float() @ dq["o"].t()).to(dtype))
        close(mid, fd.swiglu(*(y.float() @ dq["gu"].t()).to(dtype).chunk(2, -1)))
        want, wstream = fd.add_rms_norm(fd.rms_norm(out, norms[1], 1e-5), x, norms[2], 1e-5)
        torch.testing.assert_close(y.float(), want.float(), rtol=4 * tol["rtol"], atol=4 * tol["atol"])
        torch.testing.assert_close(stream.float(), wstream.float(), rtol=4 * tol["rtol"], atol=4 * tol["atol"])
        assert bool(torch.isfinite(last).all()) and bool(torch.isfinite(stream2).all())


@pytest.mark.parametrize("m", [1, 6])
def test_the_decode_step_in_four_bits(m):
    """The step's operators in its order give what its graph gives, replay for replay; a token of the cache that changes
    changes them."""
    from fused_decode.decode_step import DecodeStep

    ds = DecodeStep(m=m, layers=2, h=512, i=768, seed=3, weights="fp4", context=300)
    eager = ds.step().clone()
    assert bool(torch.isfinite(eager).all()) and ds.weight_bytes == 2 * ((768 * 512 + 512 * 512 + 3 * 512 * 768) * 17 // 32
                                                                         + 4 * 512 * 2)
    for _ in range(3):
        assert torch.equal(ds.replay(), eager)
        assert torch.equal(ds.step(), eager)
    ds.w[0]["cache"].v[0, :, 7] ^= 0x77
    assert not torch.equal(ds.replay(), eager)
