"""CPU-only checks of the operators between the projections: the packed argument records match the C structs, the rotary
speeds match the definition, the definitions used by the GPU tests agree with differently written ones, and every refusal
comes back as an error with a message (no GPU needed)."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from attention_cases import attention64, norm64, rotate64, speeds
from q27b200.attention import ATTENTION, Attention, KvCache
from q27b200.q27lib import call
from q27b200.rotary import QK_ROPE, Rotary, qk_norm_rope, rope

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fields(struct):
    text = open(os.path.join(ROOT, "include", "q27b200", "capi.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        names += [re.sub(r".*[\s*]", "", part.strip()) for part in decl.split(",") if part.strip()]
    return names


@pytest.mark.skipif(not shutil.which("gcc"), reason="needs a C compiler")
@pytest.mark.parametrize("struct,packer", [("q27b_qk_rope", QK_ROPE), ("q27b_attention", ATTENTION)])
def test_packed_records_match_the_header(tmp_path, struct, packer):
    names = fields(struct)
    values = packer.unpack(bytes(packer.size))
    assert len(values) == len(names)
    lines = "".join(f'printf("%zu\\n", offsetof({struct}, {n}));' for n in names)
    (tmp_path / "o.c").write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "q27b200/capi.h"\nint main(void) {{ printf("%zu\\n", sizeof({struct})); {lines} return 0; }}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "o.c"), "-o", str(tmp_path / "o")], check=True)
    size, *offsets = map(int, subprocess.run([str(tmp_path / "o")], capture_output=True, text=True, check=True).stdout.split())
    assert size == packer.size
    for i, at in enumerate(offsets):  # a one in field i lies where the compiler puts field i
        one = packer.pack(*[(1.0 if isinstance(v, float) else 1) if k == i else v for k, v in enumerate(values)])
        where = [k for k, byte in enumerate(one) if byte]
        assert where and at <= where[0] < at + 4, names[i]


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 32.0)])
@pytest.mark.parametrize("rot,base", [(128, 1e6), (64, 10000.0), (8, 500.0)])
def test_rotary_speeds(rot, base, scaling, factor):
    r = Rotary(rot, base, scaling=scaling, factor=factor, original_len=8192, device="cpu")
    w, a = speeds(rot, base, scaling, factor, 8192)
    got = torch.tensor([(t % (1 << 64)) / 2.0 ** 64 for t in r.turns.tolist()], dtype=torch.float64) * (2 * torch.pi)
    assert r.turns.shape == (rot // 2,) and torch.allclose(got, w, rtol=1e-14, atol=1e-18) and abs(r.amplitude - a) < 1e-6
    assert Rotary(rot, base, amplitude=0.5, device="cpu").amplitude == 0.5


def test_the_definitions_agree_with_others():
    torch.manual_seed(1)
    x, pos = torch.randn(5, 3, 16, dtype=torch.float64), torch.tensor([0, 1, 7, 100, 12345])
    w, _ = speeds(8, 100.0)
    for inter in (False, True):
        y, _ = rotate64(x, pos, w, 1.0, inter)
        z = x[..., :8].unflatten(-1, (4, 2)) if inter else x[..., :8].unflatten(-1, (2, 4)).transpose(-1, -2)
        t = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones(5, 1, 4, dtype=torch.float64), (pos[:, None] * w)[:, None])
        t = torch.view_as_real(t)
        t = t.flatten(-2) if inter else t.transpose(-1, -2).flatten(-2)
        assert torch.allclose(y, torch.cat([t, x[..., 8:]], -1), atol=1e-12)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))  # a rotation
    weight = torch.randn(16, dtype=torch.float64)
    assert torch.allclose(norm64(x, weight, 0.0, False), torch.nn.functional.rms_norm(x, (16,), weight, eps=0.0))
    q, k, v = torch.randn(4, 6, 8), torch.randn(9, 2, 8), torch.randn(9, 2, 8)
    out, lse, bound, _ = attention64(q, k, v, 4, 9, 3, 1, 0.3)
    for i in range(4):
        for h in range(6):
            p = 5 + i
            js = [j for j in range(9) if j <= p and (j > p - 3 or j < 1)]
            s = torch.stack([0.3 * (q[i, h].double() @ k[j, h // 3].double()) for j in js])
            assert torch.allclose(out[i, h], sum(a * v[j, h // 3].double() for a, j in zip(torch.softmax(s, 0), js)), atol=1e-12)
            assert torch.allclose(lse[i, h], torch.logsumexp(s, 0))
    assert attention64(q, k[:2], v[:2], 4, 2, 0, 0, 1.0)[1][:2].isneginf().all()  # positions -2 and -1 see nothing


# ---- refusals: addresses that are never touched ----------------------------------------------------------------------


def rope_record(**change):
    names = fields("q27b_qk_rope")
    r = dict.fromkeys(names, 0)
    r.update(T=4, q_heads=2, k_heads=1, head_dim=64, rot_dim=64, in_dtype=1, out_dtype=1, pos64=1, eps=1e-6, amplitude=1.0, positions=1 << 20, turns=1 << 20,
             q=1 << 20, q_ld_token=128, q_ld_head=64, k=1 << 20, k_ld_token=64, k_ld_head=64, q_out=1 << 21, q_out_ld_token=128, q_out_ld_head=64,
             k_out=1 << 21, k_out_ld_token=64, k_out_ld_head=64)
    assert set(change) <= set(names)
    r.update(change)
    return QK_ROPE.pack(*[r[n] for n in names])


@pytest.mark.parametrize("change,message", [
    ({"head_dim": 260}, "head_dim"), ({"head_dim": 12}, "head_dim"), ({"rot_dim": 72}, "rot_dim"), ({"rot_dim": 4}, "rot_dim"), ({"rot_dim": 0}, "rot_dim"),
    ({"T": -1}, "bad counts"), ({"q_heads": 0}, "bad counts"), ({"k_heads": -1}, "bad counts"), ({"in_dtype": 3}, "unknown type"), ({"out_dtype": -1}, "unknown type"),
    ({"positions": 0}, "positions"), ({"turns": 0}, "frequencies"), ({"q": 0}, "q and q_out"), ({"q": (1 << 20) + 4}, "q and q_out"), ({"q_ld_head": 66}, "q and q_out"),
    ({"q_out": 0}, "q and q_out"), ({"k": 0}, "k must not be null"), ({"k_out": 0}, "k_out must not be null"), ({"k_ld_token": 2}, "k must not be null"),
    ({"q_weight": 1 << 20}, "both weights"), ({"q_weight": (1 << 20) + 2, "k_weight": 1 << 20}, "weights must be aligned"),
    ({"q_weight": 1 << 20, "k_weight": 1 << 20, "eps": -1.0}, "eps"), ({"v": 1 << 20, "v_ld_token": 64, "v_ld_head": 64}, "v goes into the cache"),
    ({"slots": 1 << 20}, "either to k_out"), ({"slots": 1 << 20, "k_out": 0}, "cache must not be null"),
    ({"k_heads": 0}, "without key heads")])
def test_qk_norm_rope_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        call("q27b_qk_norm_rope", rope_record(**change), None)


def attention_record(**change):
    names = fields("q27b_attention")
    r = dict.fromkeys(names, 0)
    r.update(dtype=1, B=2, T=2, heads=4, kv_heads=2, head_dim=64, page_size=16, pages=9, table_width=3, max_new=1, max_kv=40, scale=0.1, table_ld=3,
             table=1 << 20, kv_lens=1 << 20, q=1 << 20, q_ld_token=256, q_ld_head=64, k_cache=1 << 20, kc_ld_page=2048, kc_ld_head=1024, kc_ld_slot=64,
             v_cache=1 << 21, vc_ld_page=2048, vc_ld_head=1024, vc_ld_slot=64, out=1 << 22, out_ld_token=256, out_ld_head=64)
    assert set(change) <= set(names)
    r.update(change)
    return ATTENTION.pack(*[r[n] for n in names])


@pytest.mark.parametrize("change,message", [
    ({"dtype": 0}, "bf16 or fp16"), ({"dtype": 7}, "bf16 or fp16"), ({"B": -1}, "bad counts"), ({"T": -2}, "bad counts"), ({"heads": 5}, "multiple of kv_heads"),
    ({"kv_heads": 0}, "multiple of kv_heads"), ({"heads": 0}, "multiple of kv_heads"), ({"head_dim": 96}, "head_dim"), ({"page_size": 48}, "page_size"), ({"page_size": 8}, "page_size"),
    ({"pages": 0}, "must not be empty"), ({"table_width": 0}, "must not be empty"), ({"table_width": 1 << 27}, "2\\^30"), ({"window": -1}, "negative"), ({"sinks": -1}, "negative"),
    ({"scale": -0.1}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"max_new": 0}, "at least 1"), ({"max_kv": 0}, "at least 1"), ({"T": 3}, "one row per sequence"), ({"table": 0}, "null table"), ({"kv_lens": 0}, "null table"),
    ({"q": 0}, "q and out"), ({"q": (1 << 20) + 8}, "q and out"), ({"out": 0}, "q and out"), ({"out_ld_head": 68}, "q and out"),
    ({"k_cache": 0}, "cache must not be null"), ({"v_cache": (1 << 20) + 2}, "cache must not be null"), ({"kc_ld_slot": 60}, "cache must not be null"), ({"vc_ld_page": 4}, "cache must not be null")])
def test_attention_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        call("q27b_paged_attention", attention_record(**change), None)


def test_workspace_refuses_and_reads_no_pointer():
    n = ctypes.c_size_t()
    with pytest.raises(RuntimeError, match="head_dim"):
        call("q27b_attention_workspace", attention_record(head_dim=32), ctypes.byref(n))
    with pytest.raises(RuntimeError, match="null"):
        call("q27b_attention_workspace", attention_record(), None)


@pytest.mark.parametrize("args", [dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, base=float("nan")), dict(rot_dim=8, scaling="linear", factor=0.5),
                                  dict(rot_dim=2, scaling="ntk", factor=2.0), dict(rot_dim=8, scaling="yarn", factor=2.0), dict(rot_dim=8, scaling="yarn", factor=2.0, original_len=10, beta_fast=1.0)])
def test_rotary_refuses(args):
    with pytest.raises(RuntimeError):
        Rotary(**args, device="cpu")
    with pytest.raises(ValueError, match="scaling"):
        Rotary(8, scaling="other", device="cpu")


def test_python_refusals():
    for args in ((4, 2, 64, 0), (4, 2, 64, -1), (4, 2, 64, None, -1), (5, 2, 64), (4, 0, 64)):
        with pytest.raises(ValueError):
            Attention(*args)
    t = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    for k, v in ((t, t[:2]), (t, t.half()), (t[0], t[0]), (t.float(), t.float()), (t.transpose(2, 3), t.transpose(2, 3))):
        with pytest.raises(ValueError):
            KvCache(k, v)
    cache = KvCache(t, t.clone())
    assert (cache.pages, cache.kv_heads, cache.page_size, cache.head_dim) == (3, 2, 16, 64)
    table = torch.tensor([[2, 0, -1]], dtype=torch.int32)
    assert cache.slots(table, torch.tensor([0, 0, 0]), torch.tensor([0, 17, 40])).tolist() == [32, 1, -8]
    q, pos, r = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.arange(2), Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA device"):
        rope(r, pos, q)
    with pytest.raises(ValueError, match="CUDA device"):
        Attention(4, 2, 64)(q, cache, table, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="must be .T, 4, 32"):
        Attention(4, 2, 32)(q, cache, table, torch.zeros(1, dtype=torch.int32))
    w = torch.zeros(64)
    for kw in (dict(v=q[:, :2]), dict(slots=pos), dict(cache=cache, k_out=q[:, :2])):
        with pytest.raises(ValueError):
            qk_norm_rope(r, pos, q, q[:, :2], w, w, **kw)
    with pytest.raises(ValueError):
        qk_norm_rope(r, pos, q, q[:, :2], w, None)
