"""Rotation by position, alone and fused with the per-head norm and the write into the paged cache, against the definition in
64 bits; the bounds are derived in attention_cases.rotation_bound."""

import pytest
import torch

from attention_cases import norm64, rotate64, rotation_bound, speeds
from q27b200.attention import KvCache
from q27b200.q27lib import device_status
from q27b200.rotary import Rotary, qk_norm_rope, rope

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def close(got, want, mag, dim, normed, what=""):
    err, bound = (got.double() - want).abs(), rotation_bound(want, mag, got.dtype, dim, normed)
    assert got.shape == want.shape and bool((err <= bound).all()), (what, float((err / bound).max()))


def stacked(T, heads, kv_heads, D, dtype):
    """q, k and v as views of one projection's rows."""
    qkv = (torch.randn(T, (heads + 2 * kv_heads) * D, device="cuda") * 1.5).to(dtype)
    q, k, v = qkv.split([heads * D, kv_heads * D, kv_heads * D], 1)
    return q.unflatten(1, (heads, D)), k.unflatten(1, (kv_heads, D)), v.unflatten(1, (kv_heads, D))


@pytest.mark.parametrize("T", [1, 2, 5, 37, 4999])
@pytest.mark.parametrize("heads,kv_heads,D,rot", [(40, 8, 128, 128), (24, 4, 256, 64), (3, 1, 64, 64), (5, 5, 80, 80), (1, 1, 8, 8), (7, 7, 200, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(T, heads, kv_heads, D, rot, interleaved):
    for dtype in TYPES if T < 40 else TYPES[1:2]:
        q, k, _ = stacked(T, heads, kv_heads, D, dtype)
        pos = torch.randint(-5, 1 << 20, (T,), device="cuda", dtype=torch.int64 if T % 2 else torch.int32)
        q1, k1 = rope(Rotary(rot, 1e6, interleaved), pos, q, k)
        w, a = speeds(rot, 1e6)
        close(q1, *rotate64(q.double(), pos, w, a, interleaved), D, False, "q")
        close(k1, *rotate64(k.double(), pos, w, a, interleaved), D, False, "k")


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 32.0), ("yarn", 1.0), ("ntk", 1.0)])
def test_rope_scalings(scaling, factor):
    q, k, _ = stacked(9, 4, 2, 128, torch.float32)
    pos = torch.tensor([0, 1, 2, 1000, 32767, 65536, 999999, 2 ** 31 - 1, 2 ** 33 + 1], device="cuda")
    r = Rotary(64, 10000.0, scaling=scaling, factor=factor, original_len=4096)
    w, a = speeds(64, 10000.0, scaling, factor, 4096)
    assert abs(r.amplitude - a) < 1e-6
    got, _ = rope(r, pos[:8], q[:8])
    close(got, *rotate64(q[:8].double(), pos[:8], w, r.amplitude, False), 128, False)
    # a position past 32 bits: the speeds' own rounding (2^-65 turns each) and fp64's in the expected angle stay below 1e-5
    far, _ = rope(r, pos[8:], q[8:])
    want, mag = rotate64(q[8:].double(), pos[8:], w, r.amplitude, False)
    assert bool(((far.double() - want).abs() <= 1e-5 * mag + 1e-6).all())
    assert rope(r, pos, q)[1] is None


def test_rope_in_place_and_strided_outputs():
    T, D = 33, 128
    q, k, _ = stacked(T, 8, 2, D, torch.bfloat16)
    pos = torch.arange(T, device="cuda") * 977
    r = Rotary(D)
    want = rope(r, pos, q, k)
    out = torch.full((8, T, D + 8), 7.0, device="cuda", dtype=torch.bfloat16)  # head-major, padded rows
    got, _ = rope(r, pos, q, q_out=out.transpose(0, 1)[..., :D])
    assert torch.equal(got, want[0]) and bool((out[..., D:] == 7).all())
    wide = torch.empty(T, 8, D, device="cuda")
    rope(r, pos, q, q_out=wide)
    assert torch.equal(wide.bfloat16(), want[0])
    back = q.clone(), k.clone()
    rope(r, pos, q, k, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert not torch.equal(back[0], q)
    assert device_status() == 0


@pytest.mark.parametrize("T", [1, 3, 33, 5000])
@pytest.mark.parametrize("heads,kv_heads,D,rot,page", [(40, 8, 128, 128, 64), (24, 4, 256, 64, 16), (6, 1, 64, 32, 128), (2, 2, 96, 96, 32)])
@pytest.mark.parametrize("src,dst", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float16)])
def test_norm_rope_into_the_cache(T, heads, kv_heads, D, rot, page, src, dst):
    q, k, v = stacked(T, heads, kv_heads, D, src)
    if T > 2:
        q[1], k[1] = 0, 0  # a row of zeros stays zeros
        q[2] *= 1e-4
    pos = torch.randint(0, 200000, (T,), device="cuda")
    inter, centred = bool(T % 2), D != 64
    qw, kw = ((torch.randn(D, device="cuda") * 0.2).to(torch.bfloat16 if D < 200 else torch.float32) for _ in range(2))
    pages = (T + page - 1) // page + 2
    kv = torch.full((pages, 2, kv_heads, page, D), float("nan"), device="cuda", dtype=dst)  # keys and values in one tensor
    cache = KvCache(kv[:, 0], kv[:, 1])
    slots = torch.randperm(pages * page, device="cuda")[:T]
    if T > 2:
        slots[0] = -1  # a padding token
    r = Rotary(rot, 5e5, inter)
    got = qk_norm_rope(r, pos, q, k, qw, kw, EPS, centred, v, cache, slots)
    w, a = speeds(rot, 5e5)
    close(got, *rotate64(norm64(q.double(), qw, EPS, centred), pos, w, a, inter), D, True, "q")
    held = slots >= 0
    page_of, at = slots[held] // page, slots[held] % page
    want, mag = rotate64(norm64(k.double(), kw, EPS, centred), pos, w, a, inter)
    close(cache.k[page_of, :, at], want[held], mag[held], D, True, "k")
    assert torch.equal(cache.v[page_of, :, at], v[held].to(dst))  # one rounding: equal bits
    rest = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    rest[page_of, at] = False
    assert bool(kv.permute(0, 3, 1, 2, 4)[rest].isnan().all())  # nothing else was written
    assert device_status() == 0
    # the same without a cache
    q2, k2 = qk_norm_rope(r, pos, q, k, qw, kw, EPS, centred, dtype=dst)
    assert torch.equal(q2, got) and torch.equal(k2[held], cache.k[page_of, :, at])


def test_token_major_cache_and_far_slots():
    """A cache kept token by token, transposed, with offsets past 2^31 elements."""
    T, Hk, D, page = 5, 2, 256, 64
    pages = (1 << 31) // (page * Hk * D) + 3
    k = torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    cache = KvCache(k.transpose(1, 2), k.transpose(1, 2))
    k[-2:] = 0
    q, kk, _ = stacked(T, 4, Hk, D, torch.bfloat16)
    kw = torch.zeros(D, device="cuda")
    slots = (pages - 1) * page + torch.tensor([3, 2, 63, 0, 1], device="cuda")
    r, pos = Rotary(D), torch.arange(T, device="cuda")
    qk_norm_rope(r, pos, q, kk, kw, kw, cache=cache, slots=slots)
    want = qk_norm_rope(r, pos, q, kk, kw, kw)[1]
    assert torch.equal(k[-1, [3, 2, 63, 0, 1]], want) and bool((k[-2] == 0).all()) and bool((k[-1, 4:63] == 0).all())


def test_a_slot_past_the_cache_is_reported_and_not_written():
    q, k, v = stacked(2, 2, 1, 64, torch.bfloat16)
    cache = KvCache(*(torch.zeros(3, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    w, r = torch.zeros(64, device="cuda"), Rotary(64)
    assert device_status() == 0
    inner = KvCache(cache.k[:2], cache.v[:2])  # the third page is behind this cache's end
    qk_norm_rope(r, torch.arange(2, device="cuda"), q, k, w, w, v=v, cache=inner, slots=torch.tensor([32, 5], device="cuda"))
    assert device_status() == 9 and device_status() == 0
    assert bool((cache.k[2] == 0).all()) and bool((cache.k[0, 0, 5] != 0).any())


def test_no_tokens_and_captured_calls():
    r, w = Rotary(64), torch.zeros(64, device="cuda")
    e = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert rope(r, torch.empty(0, dtype=torch.int64, device="cuda"), e, e)[0].shape == (0, 4, 64)
    q, k, _ = stacked(7, 4, 2, 64, torch.bfloat16)
    pos = torch.arange(7, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    qk_norm_rope(r, pos, q, k, w, w, q_out=q_out, k_out=k_out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qk_norm_rope(r, pos, q, k, w, w, q_out=q_out, k_out=k_out)
    pos += 100
    q.mul_(2)
    g.replay()
    want = qk_norm_rope(r, pos, q, k, w, w)
    assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1])


def test_non_finite_rows_stay_in_their_row():
    q, k, _ = stacked(6, 4, 2, 128, torch.bfloat16)
    q[2, 1, 5], q[3, 0, 9] = float("nan"), float("inf")
    r, pos, w = Rotary(128), torch.arange(6, device="cuda"), torch.zeros(128, device="cuda")
    got, _ = qk_norm_rope(r, pos, q, k, w, w)
    clean = torch.ones(6, 4, dtype=torch.bool, device="cuda")
    clean[2, 1] = clean[3, 0] = False
    assert bool(got[clean].isfinite().all()) and bool(got[2, 1].isnan().all()) and bool(got[3, 0].isnan().any())
