"""The operators together, as a layer uses them: prompts, chunks, verified tokens and single tokens of a ragged batch through one
cache against the definition in 64 bits; the layer (linear.Fp4Attention) against its steps called one by one."""

import pytest
import torch

from attention_cases import attention64, norm64, rotate64, rotation_bound, speeds
from q27b200.attention import Attention, KvCache
from q27b200.linear import Fp4Attention, Fp4Linear
from q27b200.q27lib import device_status
from q27b200.rotary import Rotary, qk_norm_rope, rope

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("heads,kv_heads,D,rot,page", [(10, 2, 128, 128, 32), (6, 1, 256, 64, 64), (8, 8, 64, 64, 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 5)])
def test_a_batch_grows_through_one_cache(heads, kv_heads, D, rot, page, window, sinks):
    """Three sequences take their tokens in steps of different sizes; every step's result must be that of its tokens over all
    keys and values so far, whatever kernel it went through."""
    dtype = torch.bfloat16
    steps = [(300, 0, 17), (1, 40, 1), (1, 1, 1), (16, 129, 3), (1, 1, 0), (2, 1, 16), (90, 3, 200)]
    B, longest = 3, [sum(s[b] for s in steps) for b in range(3)]
    width = max(longest) // page + 1
    table = torch.randperm(B * width, device="cuda").int().view(B, width)
    shape = (B * width, kv_heads, page, D)
    cache = KvCache(*(torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2)))
    rotary, layer = Rotary(rot, 1e6), Attention(heads, kv_heads, D, window, sinks)
    qw, kw = (torch.randn(D, device="cuda") * 0.2 for _ in range(2))
    w, a = speeds(rot, 1e6)
    length = [0] * B
    held = [[torch.empty(0, kv_heads, D, dtype=dtype, device="cuda") for _ in range(2)] for _ in range(B)]
    for step in steps:
        T = sum(step)
        qkv = (torch.randn(T, (heads + 2 * kv_heads) * D, device="cuda") * 1.5).to(dtype)
        q, k, v = qkv.unflatten(1, (-1, D)).split([heads, kv_heads, kv_heads], 1)
        sequence = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(step, device="cuda"))
        positions = torch.cat([torch.arange(length[b], length[b] + step[b], device="cuda") for b in range(B)])
        q_out = qk_norm_rope(rotary, positions, q, k, qw, kw, EPS, v=v, cache=cache, slots=cache.slots(table, sequence, positions))
        length = [n + s for n, s in zip(length, step)]
        begin = [0, step[0], step[0] + step[1], T]
        out = layer(q_out, cache, table, torch.tensor(length, dtype=torch.int32, device="cuda"), torch.tensor(begin, dtype=torch.int32, device="cuda"), max(step))
        want, mag = rotate64(norm64(k.double(), kw, EPS, True), positions, w, a, False)
        for b in range(B):
            rows = slice(begin[b], begin[b + 1])
            j = torch.arange(length[b] - step[b], length[b], device="cuda")
            new_k, new_v = (t[table[b, j // page].long(), :, j % page] for t in (cache.k, cache.v))
            assert bool(((new_k.double() - want[rows]).abs() <= rotation_bound(want[rows], mag[rows], dtype, D, True)).all())
            assert torch.equal(new_v, v[rows])
            held[b] = [torch.cat([held[b][0], new_k]), torch.cat([held[b][1], new_v])]
            o, _, bound, _ = attention64(q_out[rows], *held[b], step[b], length[b], window or 0, sinks, D ** -0.5)
            assert bool(((out[rows].double() - o).abs() <= bound).all()), (step, b)
    assert device_status() == 0


def linear(n, k, scale, seed):
    g = torch.Generator().manual_seed(seed)
    return Fp4Linear.from_float(torch.randn(n, k, generator=g) * 0.05, scale)


@pytest.mark.parametrize("M,split", [(7, (1, 6)), (128, (100, 28)), (200, (150, 50))])
@pytest.mark.parametrize("norm", [True, False])
def test_the_layer_is_its_steps(M, split, norm):
    hidden, heads, kv_heads, D, page = 512, 4, 1, 128, 16
    q, k, v = linear(heads * D, hidden, 0.01, 1), linear(kv_heads * D, hidden, 0.01, 2), linear(kv_heads * D, hidden, 0.01, 3)
    o = linear(hidden, heads * D, 0.002, 4)
    weights = [torch.randn(D, device="cuda") * 0.2 for _ in range(2)] if norm else [None, None]
    rotary = Rotary(D)
    layer = Fp4Attention(q, k, v, o, D, rotary, *weights, window=90, sinks=2)
    x, residual = torch.randn(M, hidden, device="cuda").bfloat16(), torch.randn(M, hidden, device="cuda")
    width = max(split) // page + 1
    table = torch.arange(2 * width, dtype=torch.int32, device="cuda").view(2, width)
    caches = [KvCache(*(torch.zeros(2 * width, kv_heads, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))) for _ in range(2)]
    positions = torch.cat([torch.arange(n, device="cuda") for n in split])
    slots = caches[0].slots(table, torch.repeat_interleave(torch.arange(2, device="cuda"), torch.tensor(split, device="cuda")), positions)
    lens, begin = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (split, (0, split[0], M)))
    got = layer(x, positions, caches[0], slots, table, lens, begin, max(split), residual=residual)
    parts = [p(x).unflatten(1, (-1, D)) for p in (q, k, v)]
    if norm:
        qr = qk_norm_rope(rotary, positions, parts[0], parts[1], *weights, v=parts[2], cache=caches[1], slots=slots)
    else:
        qr = rope(rotary, positions, parts[0], parts[1], v=parts[2], cache=caches[1], slots=slots)
    # (stacked or not, a projection's row has the same bits: the split of the sums depends on the weight's shape, so only many rows are asked for it)
    if M > 128:
        assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    else:
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):  # two roundings of sums that differ by fp32 steps
            assert bool(((a.float() - b.float()).abs() <= 2 ** -6 * b.float().abs() + 1e-3).all())
    y = Attention(heads, kv_heads, D, 90, 2)(qr, caches[1], table, lens, begin, max(split))
    want = o(y.flatten(1), out_dtype=torch.float32, residual=residual)
    # the output projection quantises its input to four bits: a step of one rounding there moves an output by a few percent of its spread
    assert float((got - want).norm() / (want - residual).norm()) < (1e-6 if M > 128 else 0.1)
    assert layer(x[:0], positions[:0], caches[0], slots[:0], table, lens, begin).shape == (0, hidden)
    assert device_status() == 0
