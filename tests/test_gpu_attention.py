"""Attention over the paged cache against its definition in 64 bits. Every cache is full of NaN outside the tokens that count,
every table entry that no row needs names no page; the bounds are derived in attention_cases.attention64."""

import math

import pytest
import torch

from attention_cases import attention64
from q27b200.attention import Attention, KvCache
from q27b200.q27lib import device_status

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences of (new, length) with random keys and values in pages of a NaN-filled cache."""

    def __init__(self, seqs, heads, kv_heads, D, page, window=0, sinks=0, dtype=torch.bfloat16, std=1.5, form="pages", extra_rows=0, spare=2):
        self.seqs, self.window, self.sinks = seqs, window, sinks
        self.heads, self.kv_heads, self.D, self.page = heads, kv_heads, D, page
        need = [(n + page - 1) // page for _, n in seqs]
        pages, width = sum(need) + spare, max(max(need), 1) + 1
        nan = float("nan")
        if form == "pages":
            k, v = (torch.full((pages, kv_heads, page, D), nan, device="cuda", dtype=dtype) for _ in range(2))
        elif form == "tokens":  # token by token, transposed
            k, v = (torch.full((pages, page, kv_heads, D), nan, device="cuda", dtype=dtype).transpose(1, 2) for _ in range(2))
        else:  # keys and values in one tensor, padded
            kv = torch.full((pages, 2, kv_heads, page, D + 8), nan, device="cuda", dtype=dtype)
            k, v = kv[:, 0, ..., :D], kv[:, 1, ..., :D]
        self.cache = KvCache(k, v)
        order = torch.randperm(pages, device="cuda")
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32, device="cuda")
        self.table[:, -1] = 1 << 30
        self.q = (torch.randn(sum(n for n, _ in seqs) + extra_rows, heads, D, device="cuda") * std).to(dtype)
        self.keys, self.values, used = [], [], 0
        for b, (new, length) in enumerate(seqs):
            K, V = (torch.randn(length, kv_heads, D, device="cuda").to(dtype) for _ in range(2))
            self.keys.append(K), self.values.append(V)
            mine = order[used:used + need[b]]
            used += need[b]
            j = torch.arange(length, device="cuda")
            k[mine[j // page], :, j % page], v[mine[j // page], :, j % page] = K, V
            self.table[b, :need[b]] = mine.int()
            if window:  # pages that no row sees: given back, and full of NaN
                low = length - new - window + 1
                for i in range(need[b]):
                    if i * page >= sinks and (i + 1) * page <= low:
                        self.table[b, i] = -1 if i % 2 else 1 << 29
                        k[mine[i]] = v[mine[i]] = nan
        self.kv_lens = torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda")
        self.q_begin = torch.tensor([sum(n for n, _ in seqs[:b]) for b in range(len(seqs) + 1)], dtype=torch.int32, device="cuda")

    def layer(self, scale=None):
        return Attention(self.heads, self.kv_heads, self.D, self.window or None, self.sinks, scale)

    def run(self, rows=True, scale=None, **kw):
        if rows:
            kw.setdefault("max_new", max(n for n, _ in self.seqs))
            kw.setdefault("max_kv", max(n for _, n in self.seqs))
        return self.layer(scale)(self.q, self.cache, self.table, self.kv_lens, self.q_begin if rows else None, **kw)

    def check(self, out, lse=None, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        at = 0
        for b, (new, length) in enumerate(self.seqs):
            want, wl, bound, lb = attention64(self.q[at:at + new], self.keys[b], self.values[b], new, length, self.window, self.sinks, scale)
            err = (out[at:at + new].double() - want).abs()
            assert bool((err <= bound).all()), (b, new, length, float((err / bound).nan_to_num(nan=math.inf).max()))
            if lse is not None:
                got = lse[at:at + new].double()
                assert torch.equal(got.isneginf(), wl.isneginf()), (b, new, length)
                fine = ~wl.isneginf()
                assert bool(((got - wl).abs()[fine] <= lb[fine]).all()), (b, new, length, float(((got - wl).abs() / lb)[fine].max()))
            at += new
        assert device_status() == 0


SHAPES = [(40, 8, 128), (24, 4, 256), (16, 16, 64), (12, 1, 128), (7, 7, 128), (64, 8, 64), (1, 1, 256), (48, 2, 64)]


@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (100, 0), (64, 4), (37, 130), (300, 64), (1 << 30, 3)])
def test_one_token_per_sequence(heads, kv_heads, D, page, window, sinks):
    dtype = torch.float16 if page in (16, 64) else torch.bfloat16
    b = Batch([(1, n) for n in (1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1111)], heads, kv_heads, D, page, window, sinks, dtype)
    lse = torch.empty(len(b.seqs), heads, device="cuda")
    b.check(b.run(rows=False, lse=lse), lse)
    b.check(b.run(rows=True, lse=lse), lse)


@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (70, 3), (129, 64), (3, 300)])
def test_a_few_tokens_per_sequence(heads, kv_heads, D, page, window, sinks):
    seqs = [(2, 2), (3, 1), (16, 700), (5, 64), (1, 300), (0, 40), (4, 0), (8, 129), (16, 16), (9, 1025)]
    b = Batch(seqs, heads, kv_heads, D, page, window, sinks, torch.bfloat16 if page == 16 else torch.float16)
    lse = torch.empty(b.q.shape[0], heads, device="cuda")
    b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 64), (torch.float16, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (128, 1), (200, 130), (5, 0)])
def test_prompts_and_chunks(heads, kv_heads, D, dtype, page, window, sinks):
    seqs = [(17, 17), (129, 129), (300, 300), (64, 900), (255, 256), (1, 777), (130, 100), (0, 0), (33, 1500)]
    b = Batch(seqs, heads, kv_heads, D, page, window, sinks, dtype)
    lse = torch.empty(b.q.shape[0], heads, device="cuda")
    b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1000, 100)])
@pytest.mark.parametrize("heads,kv_heads,D", [(10, 2, 128), (6, 1, 256), (4, 4, 64)])
def test_long(heads, kv_heads, D, window, sinks):
    for seqs in ([(1, 40001)], [(7, 33000), (1, 5)], [(1025, 9000)], [(4100, 4100)]):
        b = Batch(seqs, heads, kv_heads, D, 64, window, sinks)
        b.check(b.run())


@pytest.mark.parametrize("form", ["tokens", "combined"])
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 77)], [(6, 300), (2, 77)], [(140, 300), (30, 77)]])
def test_strides(form, seqs):
    b = Batch(seqs, 10, 2, 128, 32, 90, 5, form=form)
    T = b.q.shape[0]
    wide = torch.randn(T, 14, 128, device="cuda", dtype=torch.bfloat16)  # q inside the stacked projection's rows
    wide[:, :10] = b.q
    b.q = wide[:, :10]
    whole = torch.full((10, T, 136), 9.0, device="cuda", dtype=torch.bfloat16)
    out = whole.transpose(0, 1)[..., :128]  # head-major, padded
    b.check(b.run(out=out))
    assert bool((whole[..., 128:] == 9).all())
    table = torch.full((len(seqs), 2 * b.table.shape[1]), -7, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    before = out.clone()
    b.table = table[:, :b.table.shape[1]]  # rows of a wider table
    assert torch.equal(b.run(), before)


@pytest.mark.parametrize("seqs", [[(1, 300), (3, 77)], [(140, 300), (2, 77)], [(400, 400)]])
def test_rows_in_no_sequence_are_left_alone(seqs):
    b = Batch(seqs, 10, 2, 128, 32, extra_rows=5)
    b.q[-5:] = float("nan")
    out = torch.full_like(b.q, 3.0)
    lse = torch.full((b.q.shape[0], 10), 4.0, device="cuda")
    b.check(b.run(out=out, lse=lse), lse)
    assert bool((out[-5:] == 3).all()) and bool((lse[-5:] == 4).all())
    # rows before the first sequence, too
    b.q_begin += 2
    b.q[2:] = b.q[:-2].clone()
    out.fill_(3.0)
    b.run(out=out)
    b.q = b.q[2:]
    assert bool((out[:2] == 3).all()) and bool((out[-3:] == 3).all())
    b.check(out[2:])


@pytest.mark.parametrize("seqs", [[(1, 900), (1, 20)], [(6, 900), (1, 20)], [(200, 900), (3, 20), (1, 70)]])
def test_the_hints_steer_only_the_split(seqs):
    b = Batch(seqs, 10, 2, 128, 32, 300, 4)
    for new in (1, 7, 1000):
        for kv in (1, 64, 100000):
            b.check(b.run(max_new=new, max_kv=kv))
    b.check(b.layer()(b.q, b.cache, b.table, b.kv_lens, b.q_begin))


@pytest.mark.parametrize("std,scale", [(30.0, None), (1.5, 3.0), (1.5, 0.0)])
@pytest.mark.parametrize("seqs", [[(1, 3000)], [(5, 500)], [(300, 700)]])
def test_peaked_and_flat_scores(std, scale, seqs):
    b = Batch(seqs, 8, 2, 128, 64, std=std)
    lse = torch.empty(b.q.shape[0], 8, device="cuda")
    b.check(b.run(scale=scale, lse=lse), lse, scale)


@pytest.mark.parametrize("seqs", [[(1, 3000)], [(5, 2900)], [(300, 2900)]])
def test_a_maximum_that_keeps_growing(seqs):
    """Keys whose scores rise from the first to the last, so that every tile brings a new maximum; and the other way round."""
    for sign in (1.0, -1.0):
        b = Batch(seqs, 2, 1, 128, 64)
        n = seqs[0][1]
        b.q.fill_(1.0)
        b.keys[0][:] = (torch.linspace(-20, 20, n, device="cuda") * sign)[:, None, None].bfloat16()
        j = torch.arange(n, device="cuda")
        b.cache.k[b.table[0, j // 64].long(), :, j % 64] = b.keys[0]
        lse = torch.empty(b.q.shape[0], 2, device="cuda")
        b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("seqs", [[(1, 700), (1, 64)], [(4, 700), (2, 100)], [(150, 700), (90, 90)]])
def test_non_finite_queries_and_masked_keys(seqs):
    """A NaN or an infinity in one query stays in that row; in a key that a row does not see it does not reach the row."""
    b = Batch(seqs, 4, 2, 128, 64, window=50, sinks=3)
    b.q[1, 2, 7] = float("nan")
    out = b.run()
    clean = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    clean[1, 2] = False
    assert bool(out[clean].isfinite().all()) and bool(out[1, 2].isnan().all())
    b = Batch(seqs, 4, 2, 128, 64, window=50, sinks=3)
    want = b.run()
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        c = Batch(seqs, 4, 2, 128, 64, window=50, sinks=3)
        c.q, c.table, c.keys, c.values = b.q, b.table, b.keys, b.values
        c.cache = KvCache(b.cache.k.clone(), b.cache.v.clone())
        at = 0
        for i, (new, length) in enumerate(seqs):  # the last key: only the last row sees it
            j = length - 1
            c.cache.k[c.table[i, j // 64].long(), :, j % 64] = bad
        out = c.run()
        for new, _ in seqs:
            assert torch.equal(out[at:at + new - 1], want[at:at + new - 1])
            at += new


@pytest.mark.parametrize("seqs", [[(1, 700), (1, 64)], [(4, 700), (2, 100)], [(150, 700), (90, 90)]])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_infinite_or_nan_score_makes_the_row_nan(seqs, D, bad):
    """At every place of a tile, whichever way its exponential is taken: one key of the first sequence, seen by all its rows."""
    for j in (0, 1, 2, 3, 5, 37, 66, 127, 130, 300):
        b = Batch(seqs, 4, 2, D, 64)
        b.q.abs_()
        b.cache.k[b.table[0, j // 64].long(), :, j % 64] = bad
        out = b.run()
        assert bool(out[:seqs[0][0]].isnan().all()) and bool(out[seqs[0][0]:].isfinite().all()), j


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements (one tensor for keys and values), sequences in its last pages."""
    D, page, Hk = 128, 64, 8
    pages = (1 << 31) // (D * page * Hk) + 40
    k = torch.empty(pages, Hk, page, D, dtype=torch.bfloat16, device="cuda")
    k[-40:].normal_()
    for new in (1, 6, 200):
        b = Batch([(new, 1000)], 16, Hk, D, page)
        b.cache = KvCache(k, k)
        b.table[0, :16] = torch.arange(pages - 1, pages - 17, -1, device="cuda")
        j = torch.arange(1000, device="cuda")
        b.keys[0] = b.values[0] = k[b.table[0, j // page].long(), :, j % page]
        b.check(b.run())


@pytest.mark.parametrize("seqs", [[(1, 900), (1, 20), (1, 5000)], [(6, 900), (1, 20)], [(200, 900), (3, 20), (1, 70)], [(700, 5000)]])
def test_the_same_bits_every_time_and_on_every_stream(seqs):
    b, other = Batch(seqs, 40, 8, 128, 64, 3000, 4), Batch(seqs, 40, 8, 128, 64, 3000, 4)
    want, theirs = b.run(), other.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {}
    for turn in range(20):  # two callers at once
        for i, (s, x) in enumerate(zip(streams, (b, other))):
            with torch.cuda.stream(s):
                got[turn, i] = x.run()
    torch.cuda.synchronize()
    for (_, i), out in got.items():
        assert torch.equal(out, (want, theirs)[i])


@pytest.mark.parametrize("seqs", [[(1, 900), (1, 20), (1, 2000)], [(6, 900), (2, 20)], [(200, 900), (3, 20), (1, 70)]])
def test_captured_calls_follow_what_the_device_holds(seqs):
    """Two graphs of one layer replayed at once; the lengths, the table, the rows and q change between replays."""
    graphs = []
    for _ in range(2):
        b = Batch(seqs, 10, 2, 128, 32)
        b.window, b.sinks = 700, 4  # (with every page kept, so that shorter lengths find theirs)
        b.out = torch.empty_like(b.q)
        b.run(out=b.out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(out=b.out)
        graphs.append((g, b))
    streams = [torch.cuda.Stream() for _ in graphs]
    for change in range(3):
        for _, b in graphs:
            if change:
                b.q.normal_()
                b.seqs = [(new, max(length - 61, 0)) for new, length in b.seqs]
                b.kv_lens.copy_(torch.tensor([n for _, n in b.seqs], dtype=torch.int32))
                b.keys = [k[:n] for k, (_, n) in zip(b.keys, b.seqs)]
                b.values = [v[:n] for v, (_, n) in zip(b.values, b.seqs)]
            b.out.fill_(float("nan"))
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, b in graphs:
            b.check(b.out)


def test_bad_pages_and_lengths_are_reported():
    for seqs in ([(1, 200), (1, 30)], [(5, 200), (2, 30)], [(150, 200), (2, 30)]):
        b = Batch(seqs, 4, 2, 64, 16)
        good = b.run()
        assert device_status() == 0
        for bad in (-1, b.cache.pages, 1 << 30):
            keep = b.table[0, 3].clone()
            b.table[0, 3] = bad
            out = b.run()
            assert device_status() == 10
            at = seqs[0][0]
            assert torch.equal(out[at:], good[at:])  # the other sequence is not touched by it
            b.table[0, 3] = keep
        b.kv_lens[0] = 100000  # past the table
        out = b.run()
        assert device_status() == 10 and torch.equal(out[seqs[0][0]:], good[seqs[0][0]:])
        assert device_status() == 0


@pytest.mark.parametrize("new", [1, 5, 100])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 1, 128), (6, 2, 256), (3, 1, 64)])
def test_a_cache_of_one_page_and_pages_shared_by_sequences(new, heads, kv_heads, D):
    b = Batch([(new, 128)], heads, kv_heads, D, 128, spare=0)
    assert b.cache.pages == 1
    want = b.run()
    b.check(want)
    # two sequences over the same pages, one of them a token shorter
    both = b.layer()(torch.cat([b.q, b.q]), b.cache, b.table.expand(2, -1), torch.tensor([128, 127], dtype=torch.int32, device="cuda"),
                     torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda"), new)
    b.check(both[:new])
    o, _, bound, _ = attention64(b.q, b.keys[0][:127], b.values[0][:127], new, 127, 0, 0, D ** -0.5)
    assert bool(((both[new:].double() - o).abs() <= bound).all())


def test_nothing_to_do():
    b = Batch([(1, 10)], 4, 2, 64, 16)
    layer = b.layer()
    e = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert layer(e, b.cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), none).shape == (0, 4, 64)
    assert layer(e, b.cache, b.table, b.kv_lens, torch.zeros(2, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    # crooked row bounds read and write nothing outside q
    out = torch.full((1, 4, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    for begin in ([0, -3], [5, 9], [-4, 0], [1, 0]):
        layer(b.q, b.cache, b.table, b.kv_lens, torch.tensor(begin, dtype=torch.int32, device="cuda"), out=out)
        assert bool((out == 5).all())
