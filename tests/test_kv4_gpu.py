"""The 4-bit key/value cache on the GPU against plain 64-bit forms (kv4_reference)."""
from __future__ import annotations

import math

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gcnasm_b200 import kv4
    return kv4


class Case:
    """A cache of random codes whose pages lie in random order; slots that no sequence uses, and tokens
    past a sequence's end, hold bytes that would spoil a result (scale 255, the largest codes)."""

    def __init__(self, lens, hk, D, page, seed=0, low=121, high=130):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hk, self.D, self.page = list(lens), hk, D, page
        width = max(1, max((n + page - 1) // page for n in lens)) + 1
        pages = width * len(lens) + 3
        shape = (pages, hk, page)
        perm = torch.randperm(pages, generator=g)[:width * len(lens)]
        self.table = perm.view(len(lens), width).to(torch.int32)
        self.cpu = {}
        for name in ("k", "v"):
            codes = torch.full((*shape, D // 2), 0x77, dtype=torch.uint8)
            scale = torch.full((*shape, D // 32), 255, dtype=torch.uint8)
            for b, n in enumerate(lens):
                if n == 0:
                    continue
                j = torch.arange(n)
                p, s = self.table[b][j // page].long(), j % page
                codes[p, :, s] = torch.randint(0, 256, (n, hk, D // 2), generator=g, dtype=torch.int16).to(torch.uint8)
                scale[p, :, s] = torch.randint(low, high, (n, hk, D // 32), generator=g, dtype=torch.int16).to(torch.uint8)
            self.cpu[name], self.cpu[name + "_scale"] = codes, scale
        self.g = g

    def gpu(self, kv4):
        d = {n: t.cuda() for n, t in self.cpu.items()}
        return kv4.KV4Cache(d["k"], d["v"], d["k_scale"], d["v_scale"])

    def ints(self, news):
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        return cu, self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda()

    def q(self, rows, heads):
        return torch.randn((rows, heads, self.D), generator=self.g).to(torch.bfloat16)


def within(got, want, tol, what):
    got = got.double().cpu()
    same = (got == want) | ((got - want).abs() <= tol)
    bad = (~same).sum().item()
    worst = ((got - want).abs() / tol.clamp(min=1e-300))[~same].max().item() if bad else 0.0
    assert not bad, f"{what}: {bad} of {same.numel()} beyond the bound, worst {worst:.3g} times"


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,hk,news,lens", [
    (16, 1, [1], [1]),
    (64, 3, [1, 1, 1], [1, 64, 65]),
    (32, 2, [5, 0, 33, 70], [5, 9, 40, 131]),
])
def test_append_then_read(kv4, D, dtype, page, hk, news, lens):
    c = Case(lens, hk, D, page, seed=D + page)
    cache = c.gpu(kv4)
    cu, table, dl, dcu = c.ints(news)
    # K and V are parts of wider rows: neither rows nor heads are contiguous
    x = (torch.randn((cu[-1], 2 * hk + 1, D + 32), generator=c.g) * torch.exp(2 * torch.randn((cu[-1], 2 * hk + 1, 1), generator=c.g))).to(dtype)
    gx = x.cuda()
    k, v = gx[:, :hk, :D], gx[:, hk + 1:, :D]
    w = kv4.alloc_weights(cache)
    w.fill_(7.0)
    one = all(n == 1 for n in news)
    kv4.append(cache, k, v, table, dl, None if one else dcu, weights=w)
    want = {n: t.clone() for n, t in c.cpu.items()}
    ww = torch.full(w.shape, 7.0)
    for b, n in enumerate(news):
        j = lens[b] - n + torch.arange(n)
        p, s = c.table[b][j // page].long(), j % page
        for name, src in (("k", x[:, :hk, :D]), ("v", x[:, hk + 1:, :D])):
            want[name][p, :, s], want[name + "_scale"][p, :, s] = R.quantise(src[cu[b]:cu[b + 1]])
        ww[p, :, s] = 0.0
    for name in want:
        assert torch.equal(getattr(cache, name).cpu(), want[name]), name
    assert torch.equal(w.cpu(), ww)
    start = dl - torch.tensor(news, dtype=torch.int32).cuda()
    rk, rv = kv4.read(cache, table, start, dcu, cu[-1])
    for b, n in enumerate(news):
        for name, got in (("k", rk), ("v", rv)):
            ref = R.tokens(want, name, c.table, b, page, lens[b])[lens[b] - n:]
            assert torch.equal(got[cu[b]:cu[b + 1]].cpu(), ref.to(torch.bfloat16)), (b, name)


def test_append_special_values(kv4):
    """Zeros, signed zeros, infinities, NaN, subnormals, the largest and smallest magnitudes, every tie."""
    D, hk = 128, 1
    rows = [torch.zeros(D), -torch.zeros(D), torch.full((D,), math.inf), torch.full((D,), math.nan),
            torch.full((D,), 1e-42), torch.full((D,), 3e38), torch.full((D,), 2.0 ** -61), torch.full((D,), 6.0 * 2.0 ** 65),
            torch.cat([torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -5.0, -6.0] + [0.0] * 20)] * 4),
            torch.cat([torch.tensor([math.nan, 1.0, -math.nan] + [0.1] * 29), torch.tensor([-math.inf, 5.0] + [1.0] * 30),
                       torch.tensor([6.0000005] + [5.0000005] * 31), torch.tensor([1e-30] * 32)])]
    x = torch.stack(rows)[:, None]
    n = len(rows)
    c = Case([n], hk, D, 16)
    cache = c.gpu(kv4)
    cu, table, dl, dcu = c.ints([n])
    kv4.append(cache, x.cuda(), -x.cuda(), table, dl, dcu)
    j = torch.arange(n)
    p, s = c.table[0][j // 16].long(), j % 16
    for name, src in (("k", x), ("v", -x)):
        codes, scale = R.quantise(src)
        assert torch.equal(getattr(cache, name + "_scale").cpu()[p, :, s], scale)
        assert torch.equal(getattr(cache, name).cpu()[p, :, s], codes)
    rk, rv = kv4.read(cache, table, torch.zeros(1, dtype=torch.int32).cuda(), dcu, n)
    assert torch.isfinite(rk.float()).all() and torch.isfinite(rv.float()).all()


def test_append_drops_what_does_not_fit(kv4):
    """More rows than tokens (positions before the start) and a length past the table are cut, not written."""
    c = Case([3, 40], 2, 64, 16)
    cache = c.gpu(kv4)
    table = c.table[:, :2].contiguous()  # 32 tokens a sequence
    x = torch.randn((15, 2, 64), generator=c.g)
    cu = torch.tensor([0, 5, 15], dtype=torch.int32)
    kv4.append(cache, x.cuda(), x.cuda(), table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), cu.cuda())
    want = {n: t.clone() for n, t in c.cpu.items()}
    for b, row, j in [(0, 2, 0), (0, 3, 1), (0, 4, 2), (1, 5, 30), (1, 6, 31)]:
        p, s = table[b][j // 16].long(), j % 16
        for name in ("k", "v"):
            want[name][p, :, s], want[name + "_scale"][p, :, s] = R.quantise(x[row])
    for name in want:
        assert torch.equal(getattr(cache, name).cpu(), want[name]), name


# ------------------------------------------------------------------ attention
def attend(kv4, c, news, heads, scale=None, one_row=False, **mask):
    cu, table, lens, dcu = c.ints(news)
    q = c.q(cu[-1], heads)
    cache = c.gpu(kv4)
    scale = c.D ** -0.5 if scale is None else scale
    out, lse = kv4.attention(q.cuda(), cache, table, lens, None if one_row else dcu, max_q=max(news), scale=scale, **mask)
    want = R.attention(q, c.cpu, c.table, c.lens, cu, c.page, scale, **mask)
    within(out, want[0], want[2], "out")
    within(lse, want[1], want[3], "lse")
    return q, cache, table, lens, dcu, out, lse, want


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hk,group", [(1, 1), (2, 4), (1, 7), (2, 8), (1, 16), (1, 40)])
def test_attention_one_token(kv4, D, hk, group):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 255, 257, 700]
    attend(kv4, Case(lens, hk, D, 32, seed=group), [1] * len(lens), hk * group, one_row=True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("news,lens", [
    ([2, 3, 4, 1], [2, 130, 400, 1]),
    ([1, 9, 0, 40, 33], [300, 9, 77, 170, 600]),
    ([150, 1, 70], [150, 513, 333]),
    ([300], [1000]),
])
@pytest.mark.parametrize("mask", [dict(), dict(window=50), dict(softcap=20.0), dict(causal=False),
                                  dict(causal=False, window=9, softcap=5.0)])
def test_attention_rows_and_masks(kv4, D, page, news, lens, mask):
    attend(kv4, Case(lens, 2, D, page, seed=len(news)), news, 6, **mask)


@pytest.mark.parametrize("group", [1, 3, 5, 8, 12])
@pytest.mark.parametrize("new", [1, 2, 5, 11, 64, 129])
def test_attention_groups_by_rows(kv4, group, new):
    """Every product of group and rows around the kernels' row tiles."""
    attend(kv4, Case([new, 3 * new + 1], 2, 64, 16, seed=group + new), [new, new], 2 * group)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,lens,mask", [
    ([1, 300, 1, 2, 1, 1], [700, 350, 1, 2, 900, 33], dict()),           # prompts and single tokens in one batch
    ([70], [2500], dict()),                                              # few rows, many steps: cut across the GPU
    ([65, 1, 1], [1500, 3000, 10], dict(window=700)),
    ([40, 200], [2000, 200], dict(softcap=15.0)),
    ([500, 0, 3], [500, 40, 1200], dict(causal=False)),
])
def test_attention_cut_and_mixed(kv4, D, news, lens, mask):
    attend(kv4, Case(lens, 1, D, 64, seed=len(lens)), news, 2, **mask)


def test_attention_many_items(kv4):
    """More (sequence, head, block) items than the GPU takes at once."""
    n = 50
    attend(kv4, Case([100 + 3 * i for i in range(n)], 8, 64, 32, seed=3), [70 + i for i in range(n)], 16)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("new", [1, 6, 200])
def test_attention_nothing_seen(kv4, D, new):
    """Rows before the sequence's start and empty sequences: zero, and -inf as the logarithm."""
    c = Case([0, new // 2, new + 3], 1, D, 16)
    *_, out, lse, want = attend(kv4, c, [new, new, new], 4)
    empty = torch.isinf(want[1])
    assert empty.any()
    assert (out.cpu()[empty] == 0).all() and (lse.cpu()[empty] == -math.inf).all()
    attend(kv4, Case([0, 5], 1, D, 16), [new, new], 4, causal=False, window=3)


@pytest.mark.parametrize("new", [1, 70])
def test_attention_scale_range(kv4, new):
    """Scales over the whole range of the format; large and negative score scales."""
    c = Case([90, 300], 1, 128, 16, low=67, high=80)
    attend(kv4, c, [new, new], 4, scale=2.0 ** 60)
    c = Case([90, 300], 1, 128, 16, low=185, high=256)
    c.cpu["k_scale"].fill_(124)
    attend(kv4, c, [new, new], 4)
    c = Case([90, 300], 1, 128, 16, low=115, high=140)
    attend(kv4, c, [new, new], 4, scale=-0.3)
    attend(kv4, c, [new, new], 4, scale=0.0)
    # scores far apart: one token takes everything
    attend(kv4, Case([90, 300], 1, 128, 16, low=135, high=140), [new, new], 4, scale=8.0)


@pytest.mark.parametrize("new", [1, 5, 100])
def test_attention_strides_and_streams(kv4, new):
    """q a slice of a fused projection, out a slice of a wider buffer, on a stream of its own."""
    c = Case([400, 222], 2, 128, 64)
    cu, table, lens, dcu = c.ints([new, new])
    x = torch.randn((2 * new, 12, 192), generator=c.g).to(torch.bfloat16)
    q = x[:, 2:10, 32:160]
    cache = c.gpu(kv4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gx = x.cuda()
    buf = torch.full((2 * new, 10, 136), 3.0, dtype=torch.bfloat16, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    out, lse = kv4.attention(gx[:, 2:10, 32:160], cache, table, lens, dcu, max_q=new, out=buf[:, 1:9, 8:], stream=side)
    side.synchronize()
    want = R.attention(q, c.cpu, c.table, c.lens, cu, 64, 128 ** -0.5)
    within(out, want[0], want[2], "out")
    within(lse, want[1], want[3], "lse")
    buf[:, 1:9, 8:] = 3.0
    assert (buf == 3.0).all()


@pytest.mark.parametrize("raw", [False, True])
def test_results_belong_to_the_stream_of_the_call(kv4, raw):
    """Memory that unfinished work of the current stream still writes is not given to a call on another."""
    c = Case([400, 222], 2, 128, 64)
    cu, table, lens, dcu = c.ints([3, 3])
    q = torch.randn((6, 8, 128), generator=c.g).to(torch.bfloat16).cuda()
    cache, start = c.gpu(kv4), torch.zeros(2, dtype=torch.int32, device="cuda")
    want = (*kv4.attention(q, cache, table, lens, dcu, max_q=3), *kv4.read(cache, table, start, dcu, 6))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy = [torch.empty_like(t) for t in want for _ in range(4)]
    torch.cuda._sleep(20_000_000)
    for t in busy:
        t.fill_(3.0)
    del busy, t
    stream = side.cuda_stream if raw else side
    got = (*kv4.attention(q, cache, table, lens, dcu, max_q=3, stream=stream),
           *kv4.read(cache, table, start, dcu, 6, stream=stream))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_is_repeatable(kv4, new):
    """Bit for bit the same in every run, with other calls between: sums are in a fixed order."""
    c = Case([3000, 1700, 50, 900], 2, 128, 32)
    q, cache, table, lens, cu, out, lse, _ = attend(kv4, c, [new] * 4, 16)
    q2 = c.q(q.shape[0], 16).cuda()
    for _ in range(5):
        kv4.attention(q2, cache, table, lens, cu, max_q=new)
        o, l = kv4.attention(q.cuda(), cache, table, lens, cu, max_q=new)
        assert torch.equal(o, out) and torch.equal(l, lse)


def test_attention_bad_pages_are_absent(kv4):
    """Tokens of pages that are not there: as if the sequence had not got them, and the status word says so."""
    from gcnasm_b200 import capi, ops
    c = Case([64, 64], 1, 64, 16)
    for new in (1, 40):
        cu, table, lens, dcu = c.ints([new, new])
        cache = c.gpu(kv4)
        q = c.q(2 * new, 2)
        bad = table.clone()
        bad[0, 1], bad[1, 0] = -1, 1 << 30
        ops.device_status()
        out, lse = kv4.attention(q.cuda(), cache, bad, lens, dcu, max_q=new, causal=False)
        assert ops.device_status() == capi.DEV_BAD_PAGE
        for b, gone in ((0, 1), (1, 0)):
            rest = Case([48], 1, 64, 16)
            rest.cpu, rest.table = c.cpu, c.table[b:b + 1, [i for i in range(4) if i != gone]]
            want = R.attention(q[b * new:(b + 1) * new], c.cpu, rest.table, [48], [0, new], 16, 0.125, causal=False)
            within(out[b * new:(b + 1) * new], want[0], want[2], "out")
            within(lse[b * new:(b + 1) * new], want[1], want[3], "lse")
        w = kv4.alloc_weights(cache)
        kv4.weights(q.cuda(), lse, cache, bad, lens, w, dcu, max_q=new, causal=False)
        assert ops.device_status() == capi.DEV_BAD_PAGE
        assert torch.isfinite(w).all() and abs(w.sum().item() - 4 * new) < 1e-3 * new
        before = cache.k.clone()
        x = torch.randn((2 * new, 1, 64), generator=c.g).cuda()
        lost = torch.full_like(table, -7)
        kv4.append(cache, x, x, lost, lens, dcu)
        assert torch.equal(cache.k, before) and ops.device_status() == capi.DEV_BAD_PAGE
        k, v = kv4.read(cache, lost, lens - new, dcu, 2 * new)
        assert (k == 0).all() and (v == 0).all() and ops.device_status() == capi.DEV_BAD_PAGE


def test_past_four_gigabytes(kv4):
    """Tokens whose byte offsets pass 2^32."""
    D, hk, page = 256, 8, 1024
    pages = (1 << 32) // (hk * page * D // 2) + 3
    cache = kv4.alloc(pages, hk, D, page)
    n = 1500
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32).cuda()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    cu = torch.tensor([0, n], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(1)
    x = torch.randn((n, 2, hk, D), generator=g).to(torch.bfloat16)
    kv4.append(cache, x[:, 0].cuda(), x[:, 1].cuda(), table, lens, cu)
    small = {"k": None, "v": None}
    for i, name in enumerate(("k", "v")):
        codes, scale = R.quantise(x[:, i])
        small[name] = torch.zeros((2, page, hk, D // 2), dtype=torch.uint8)
        small[name].view(-1, hk, D // 2)[:n] = codes
        small[name] = small[name].transpose(1, 2)
        sf = torch.zeros((2, page, hk, D // 32), dtype=torch.uint8)
        sf.view(-1, hk, D // 32)[:n] = scale
        small[name + "_scale"] = sf.transpose(1, 2)
    near = torch.tensor([[0, 1]], dtype=torch.int32)
    assert (cache.k[:3] == 0).all()
    for new in (1, 70):
        q = torch.randn((new, hk, D), generator=g).to(torch.bfloat16)
        c2 = torch.tensor([0, new], dtype=torch.int32).cuda()
        out, lse = kv4.attention(q.cuda(), cache, table, lens, c2, max_q=new)
        want = R.attention(q, small, near, [n], [0, new], page, D ** -0.5)
        within(out, want[0], want[2], "out")
        within(lse, want[1], want[3], "lse")
    w = kv4.alloc_weights(cache)
    kv4.weights(q.cuda(), lse, cache, table, lens, w, c2, max_q=new)
    assert abs(w[pages - 2:].sum().item() - new * hk) < 1e-3 * new * hk and (w[:pages - 2] == 0).all()
    to = torch.tensor([[pages - 3]], dtype=torch.int32).cuda()
    kept, _ = kv4.evict(cache, w, table, lens, 700, out_table=to)
    k, _ = kv4.read(cache, to, torch.zeros_like(lens), torch.tensor([0, 700], dtype=torch.int32).cuda(), 700)
    for h in (0, hk - 1):
        ref = R.tokens(small, "k", near, 0, page, n)[kept[0, h].cpu().long(), h].to(torch.bfloat16)
        assert torch.equal(k[:, h].cpu(), ref)


def test_in_a_graph(kv4):
    """append, attention, weights and evict captured once and replayed with other inputs."""
    c = Case([70, 333], 2, 128, 16)
    cu, table, lens, dcu = c.ints([1, 1])
    cache = c.gpu(kv4)
    w = kv4.alloc_weights(cache)
    q = c.q(2, 8).cuda()
    x = torch.randn((2, 4, 128), generator=c.g).to(torch.bfloat16).cuda()
    out_table = torch.full((2, 4), 0, dtype=torch.int32).cuda()
    free = sorted(set(range(cache.pages)) - set(c.table.flatten().tolist()))
    out_table = torch.tensor([[free[0]], [free[1]]], dtype=torch.int32).cuda()

    def step():
        kv4.append(cache, x[:, :2], x[:, 2:], table, lens, weights=w)
        out, lse = kv4.attention(q, cache, table, lens)
        kv4.weights(q, lse, cache, table, lens, w)
        return out, kv4.evict(cache, w, table, lens, 16, sink=2, recent=4, out_table=out_table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=c.g))
        x.copy_(torch.randn(x.shape, generator=c.g))
        w0 = w.clone()
        graph.replay()
        torch.cuda.synchronize()
        gout, (gkept, glens) = got[0].clone(), (got[1][0].clone(), got[1][1].clone())
        w.copy_(w0)
        out, (kept, nl) = step()
        assert torch.equal(out, gout) and torch.equal(kept, gkept) and torch.equal(nl, glens)


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hk,group,news,lens,mask", [
    (2, 4, [1, 1, 1, 1], [1, 33, 200, 515], dict()),
    (1, 7, [3, 0, 9], [3, 50, 140], dict(softcap=10.0)),
    (2, 1, [32, 40], [32, 300], dict(window=20)),
    (1, 16, [64, 5], [500, 64], dict(causal=False)),
    (1, 3, [150, 4], [100, 2], dict()),
    (2, 4, [16, 20, 1], [900, 1500, 5], dict()),
    (1, 8, [16], [2000], dict(window=300)),
    (2, 2, [40, 0, 40], [600, 300, 50], dict(softcap=8.0)),
    (1, 6, [70, 90], [400, 3000], dict(window=1000, softcap=25.0)),
    (3, 2, [30, 30], [520, 1030], dict(causal=False, window=200)),
])
def test_weights(kv4, D, hk, group, news, lens, mask):
    c = Case(lens, hk, D, 32, seed=7)
    q, cache, table, dl, dcu, out, lse, _ = attend(kv4, c, news, hk * group, **mask)
    cu = dcu.tolist()
    want = R.gathered(q, lse.cpu(), c.cpu, c.table, lens, cu, 32, D ** -0.5, **mask)
    held = torch.rand((cache.pages, hk, 32), generator=c.g)
    ref, tol = held.double().clone(), torch.zeros(held.shape, dtype=torch.float64)
    for b, (w, t) in enumerate(want):
        j = torch.arange(lens[b])
        p, s = c.table[b][j // 32].long(), j % 32
        ref[p, :, s] += w.T
        tol[p, :, s] = t.T + 2.0 ** -23 * ref[p, :, s]
    a = held.cuda()
    sums = torch.full_like(a, -1.0)
    kv4.weights(q.cuda(), lse, cache, table, dl, a, dcu, max_q=max(news), out=sums, **mask)
    assert torch.equal(a.cpu(), held)
    used = torch.zeros(held.shape, dtype=torch.bool)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        used[c.table[b][j // 32].long(), :, j % 32] = True
    assert (sums.cpu()[~used] == -1.0).all()
    within(sums.cpu()[used], ref[used], tol[used], "weights")
    kv4.weights(q.cuda(), lse, cache, table, dl, a, dcu, max_q=max(news), **mask)  # in place
    assert torch.equal(a.cpu()[used], sums.cpu()[used]) and torch.equal(a.cpu()[~used], held[~used])


# ------------------------------------------------------------------ evict
def some_weights(kind, shape, g):
    w = torch.exp(2 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 4, shape, generator=g).float()
    elif kind == "equal":
        w = torch.full(shape, 0.25)
    elif kind == "special":
        pick = torch.randint(0, 8, shape, generator=g)
        for i, v in enumerate([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-42]):
            w = torch.where(pick == i, torch.full(shape, v), w)
    return w


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("page,budget,sink,recent", [(16, 1, 0, 0), (16, 1, 1, 0), (32, 40, 4, 8), (32, 64, 0, 64), (64, 700, 3, 100), (16, 2500, 0, 5)])
def test_evict(kv4, D, kind, page, budget, sink, recent):
    lens = [0, 1, 40, 41, 700, 1025, 2600]
    hk = 2
    c = Case(lens, hk, D, page, seed=budget)
    width = (budget + page - 1) // page
    extra = width * len(lens)
    n_pages = c.cpu["k"].shape[0]
    for name in list(c.cpu):
        c.cpu[name] = torch.cat([c.cpu[name], torch.full((extra, *c.cpu[name].shape[1:]), 0xAB, dtype=torch.uint8)])
    out_table = (n_pages + torch.randperm(extra, generator=c.g)).view(len(lens), width).to(torch.int32)
    held = some_weights(kind, (n_pages + extra, hk, page), c.g)
    _, table, dl, _ = c.ints([1] * len(lens))
    want_kept = torch.full((len(lens), hk, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        for h in range(hk):
            w = held[c.table[b][j // page].long(), h, j % page].tolist()
            kp = R.kept(w, n, budget, sink, recent)
            want_kept[b, h, :len(kp)] = torch.tensor(kp, dtype=torch.int32)
    for in_place in (False, True):
        to = c.table if in_place else out_table
        want = {n: t.clone() for n, t in c.cpu.items()}
        want["w"] = held.clone()
        for b, n in enumerate(lens):
            m = min(n, budget)
            i = torch.arange(m)
            for h in range(hk):
                j = want_kept[b, h, :m].long()
                for name, src in (*c.cpu.items(), ("w", held)):
                    want[name][to[b][i // page].long(), h, i % page] = src[c.table[b][j // page].long(), h, j % page]
        cache, w, lens_gpu = c.gpu(kv4), held.cuda(), dl.clone()
        kept, new_lens = kv4.evict(cache, w, table, lens_gpu, budget, sink=sink, recent=recent,
                                   out_table=None if in_place else out_table.cuda(), out_lens=lens_gpu if in_place else None)
        assert torch.equal(kept.cpu(), want_kept)
        assert new_lens.tolist() == [min(n, budget) for n in lens]
        assert torch.equal(w.cpu().view(torch.int32), want["w"].view(torch.int32))
        for name in c.cpu:
            assert torch.equal(getattr(cache, name).cpu(), want[name]), (in_place, name)


# ------------------------------------------------------------------ refusals on a GPU's tensors
def test_refusals(kv4):
    from gcnasm_b200 import capi
    c = Case([20, 20], 2, 64, 16)
    cu, table, lens, dcu = c.ints([2, 2])
    cache = c.gpu(kv4)
    q = c.q(4, 4).cuda()
    kv = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    w = kv4.alloc_weights(cache)
    lse = torch.zeros((4, 4), device="cuda")
    with pytest.raises(ValueError):
        kv4.KV4Cache(cache.k.cpu(), cache.v, cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        kv4.KV4Cache(cache.k, cache.v[1:], cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        kv4.alloc(4, 1, 96)
    with pytest.raises(ValueError):
        kv4.append(cache, kv.half(), kv.half(), table, lens, dcu)
    with pytest.raises(ValueError):
        kv4.append(cache, kv, kv.float(), table, lens, dcu)
    with pytest.raises(ValueError):
        kv4.append(cache, kv[:, :1], kv[:, :1], table, lens, dcu)
    with pytest.raises(ValueError):
        kv4.append(cache, kv, kv, table.long(), lens, dcu)
    with pytest.raises(ValueError):
        kv4.attention(q.float(), cache, table, lens, dcu)
    with pytest.raises(ValueError):
        kv4.attention(q, cache, table, lens[:1], dcu)
    with pytest.raises(ValueError):
        kv4.attention(q, cache, table, lens, dcu[:2].contiguous())
    with pytest.raises(ValueError):
        kv4.attention(q, cache, table[:, ::2], lens, dcu)
    with pytest.raises(ValueError):
        kv4.attention(q, cache, table, lens, dcu, out=torch.empty_like(q, dtype=torch.float32))
    with pytest.raises(ValueError):
        kv4.weights(q, lse[:2], cache, table, lens, w, dcu)
    with pytest.raises(ValueError):
        kv4.weights(q, lse, cache, table, lens, w[:1], dcu)
    for call, status in [
        (lambda: kv4.attention(q, cache, table, lens), capi.B2G_ERR_INVALID_ARG),                   # rows without cu
        (lambda: kv4.attention(q[:, :3], cache, table, lens, dcu), capi.B2G_ERR_INVALID_ARG),       # heads
        (lambda: kv4.attention(q, cache, table, lens, dcu, softcap=-1.0), capi.B2G_ERR_INVALID_ARG),
        (lambda: kv4.attention(q, cache, table, lens, dcu, window=-1), capi.B2G_ERR_INVALID_ARG),
        (lambda: kv4.attention(q, cache, table, lens, dcu, scale=math.nan), capi.B2G_ERR_INVALID_ARG),
        (lambda: kv4.attention(torch.zeros((4, 4, 68), dtype=torch.bfloat16, device="cuda")[..., 2:66], cache, table, lens, dcu),
         capi.B2G_ERR_ALIGNMENT),
        (lambda: kv4.attention(q, cache, table, lens, dcu, ws=torch.zeros(8, dtype=torch.uint8, device="cuda")), capi.B2G_ERR_WORKSPACE),
        (lambda: kv4.evict(cache, w, table, lens, 0, sink=0, recent=0), capi.B2G_ERR_INVALID_ARG),
        (lambda: kv4.evict(cache, w, table, lens, 8, sink=4, recent=5), capi.B2G_ERR_INVALID_ARG),
        (lambda: kv4.evict(cache, w, table, lens, 32, sink=0, recent=0, out_table=table[:, :1].contiguous()), capi.B2G_ERR_INVALID_ARG),
    ]:
        with pytest.raises(capi.B2GError) as e:
            call()
        assert e.value.status == status
    # no rows: nothing to do
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    out, _ = kv4.attention(q[:0], cache, table, lens, none)
    assert out.shape == (0, 4, 64)
    kv4.append(cache, kv[:0], kv[:0], table, lens, none)


# ------------------------------------------------------------------ all together
def test_layer_with_eviction(kv4):
    """The demo's layer: prompts, then decode steps that thin the cache out.  Each step's output is that of
    plain 64-bit attention over what the cache held, through the same projections."""
    from gcnasm_b200 import kv4_demo, ops
    torch.manual_seed(1)
    dim, heads, kv_heads, D, budget = 256, 4, 2, 64, 48
    layer = kv4_demo.KV4Attention(torch.randn(((heads + 2 * kv_heads) * D, dim), device="cuda") * dim ** -0.5,
                                  torch.randn((dim, heads * D), device="cuda") * 0.06, heads, kv_heads, D, pages=64, page_size=16)
    seen = []

    class Spy:
        def __getattr__(self, name):
            return getattr(kv4, name)

        def attention(self, q, cache, table, lens, cu=None, **k):
            out, lse = kv4.attention(q, cache, table, lens, cu, **k)
            n = lens.tolist()
            c = cu.tolist() if cu is not None else list(range(len(n) + 1))
            cpu = {x: getattr(cache, x).cpu() for x in ("k", "v", "k_scale", "v_scale")}
            want = R.attention(q.cpu(), cpu, table.cpu(), n, c, 16, D ** -0.5)
            within(out, want[0], want[2], "out")
            within(lse, want[1], want[3], "lse")
            seen.append(n)
            return out, lse

    real, kv4_demo.kv4 = kv4_demo.kv4, Spy()
    try:
        for y, lens in kv4_demo.generate(layer, [70, 20, 33], 40, dim, budget, every=8):
            assert torch.isfinite(y).all() and y.shape[1] == dim
    finally:
        kv4_demo.kv4 = real
    assert len(seen) == 41 and seen[0] == [70, 20, 33]
    assert seen[1] == [49, 21, 34] and max(max(n) for n in seen[1:]) <= budget + 8
    assert ops.device_status() == 0
    # the weights that a sequence's tokens hold sum to at most one per query head and step seen
    assert (layer.gathered >= 0).all()
