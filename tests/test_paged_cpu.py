"""CPU: the paged-cache entry points refuse what they cannot serve, before any CUDA call."""
import ctypes

import pytest
import torch

from std_b200 import _lib, ops

A = 1 << 20  # a 16-byte aligned address that is never read


def attn(**kw):
    a = dict(q=A, k=A, v=A, table=A, cu=A, lens=A, T=4, B=1, Hq=28, Hkv=4, D=128, fp16=0, pages=8, page=16, width=4,
             causal=1, scale=0.1, out=2 * A, lse=None, ws=A, nb=1 << 40, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.load().std_paged_attn(*a.values())


@pytest.mark.parametrize("bad", [
    dict(D=96), dict(D=0), dict(T=-1), dict(B=0), dict(B=8193), dict(Hkv=0), dict(Hq=30), dict(Hq=0), dict(Hq=129, Hkv=1),
    dict(page=8), dict(page=48), dict(page=0), dict(pages=0), dict(width=0), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(table=None),
    dict(cu=None), dict(lens=None), dict(out=None), dict(out=A), dict(q=A + 8), dict(k=A + 2), dict(out=2 * A + 4),
    dict(pages=1 << 27, page=16), dict(width=1 << 27, page=16), dict(pages=1 << 22, page=256, Hkv=28)])
def test_attention_refusals(bad):
    assert attn(**bad) == 1


@pytest.mark.parametrize("bad", [dict(B=8192, Hkv=65535, Hq=65535), dict(T=1 << 30, Hkv=2000, Hq=256000)])
def test_attention_refuses_more_items_than_32_bits_count(bad):
    assert attn(pages=100, **bad) == 1


def test_attention_workspace_and_nothing_to_do():
    need = _lib.query("std_paged_attn_workspace_bytes", 128)
    assert need > 0 and _lib.query("std_paged_attn_workspace_bytes", 96) == 0
    assert attn(nb=need - 1) == 5 and attn(ws=None) == 5 and attn(ws=A + 8) == 5
    assert attn(T=0, q=None, out=None) == 0


def update(**kw):
    a = dict(past=A, new=A, table=A, nblk=A, free=A, nfree=A, B=2, width=4, page=16, pages=8, tokens=3, cu=A, kv=A,
             slots=A, pos=A, ok=A, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.load().std_paged_update(*a.values())


@pytest.mark.parametrize("bad", [
    dict(B=0), dict(B=8193), dict(width=0), dict(page=24), dict(pages=0), dict(tokens=-1), dict(past=None),
    dict(new=None), dict(table=None), dict(nblk=None), dict(free=None), dict(nfree=None), dict(cu=None), dict(kv=None),
    dict(slots=None), dict(pos=None), dict(ok=None), dict(B=8192, width=1 << 20), dict(pages=1 << 28),
    dict(width=1 << 28, B=1)])
def test_update_refusals(bad):
    assert update(**bad) == 1


def append(**kw):
    a = dict(qkv=A, T=3, Hq=28, Hkv=4, D=128, fp16=0, pos=A, slots=A, cos=A, sin=A, max_pos=9, q=A, k=A, v=A, pages=8,
             page=16, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.load().std_paged_rope_append(*a.values())


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=80), dict(max_pos=0), dict(pages=0), dict(page=20), dict(pages=1 << 28),
    dict(qkv=None), dict(pos=None), dict(slots=None), dict(cos=None), dict(sin=None), dict(q=None), dict(k=None),
    dict(v=None), dict(qkv=A + 2), dict(cos=A + 4), dict(q=A + 8), dict(k=A + 8)])
def test_append_refusals(bad):
    assert append(**bad) == 1


def test_append_nothing_to_do():
    assert append(T=0, qkv=None, q=None) == 0


def test_wrappers_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(q, k, k, i.view(1, 2), i, i[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_update(i, i, i.view(2, 1), i, i, i[:1], 16, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_rope_append(q.view(2, 64), i, i, k[0, 0], k[0, 0], q, k, k)


@pytest.mark.parametrize("scale", [2.4e38, 3e38, 3.3e38])
def test_attention_refuses_scales_that_overflow_in_log2(scale):
    assert attn(scale=scale) == 1


@pytest.mark.parametrize("fits,over", [
    (dict(T=2 ** 30 - 1, Hq=4), dict(T=2 ** 30, Hq=4)),
    (dict(width=8388603, page=256), dict(width=8388604, page=256)),            # max_blocks * page_size <= 2^31 - 1025
    (dict(pages=2 ** 21 - 2, page=256, Hkv=28), dict(pages=2 ** 22, page=256, Hkv=28)),
    (dict(pages=2396744, page=256, Hkv=28), dict(pages=2396745, page=256, Hkv=28)),  # (num_pages + 1) * Hkv * page / 8 < 2^31
])
def test_attention_limits_are_those_of_the_header(fits, over):
    """On the near side of each limit a call gets past the checks (and fails for want of
    a device), on the far side it is refused."""
    apart = dict(zip(("q", "k", "v", "table", "cu", "lens", "out", "ws"), range(1 << 44, 9 << 44, 1 << 44)))
    assert attn(**apart, **over) == 1
    if not torch.cuda.is_available():
        assert attn(**apart, **fits) not in (0, 1, 5)


# Arrays of a call, each at an address of its own (never read: without a device no call gets that far).
def apart(*names):
    return {n: (i + 1) << 44 for i, n in enumerate(names)}


UPDATE = apart("past", "new", "table", "nblk", "free", "nfree", "cu", "kv", "slots", "pos", "ok")
APPEND = apart("qkv", "pos", "slots", "cos", "sin", "q", "k", "v")
ATTN = apart("q", "k", "v", "table", "cu", "lens", "out", "lse", "ws")
SIZES = {  # bytes of each, for the sizes that update(), append() and attn() give
    "update": dict(past=8, new=8, table=32, nblk=8, free=32, nfree=4, cu=12, kv=8, slots=12, pos=12, ok=8),
    "append": dict(qkv=3 * 36 * 256, pos=12, slots=12, cos=9 * 128, sin=9 * 128, q=3 * 28 * 256, k=8 * 4 * 16 * 256,
                   v=8 * 4 * 16 * 256),
    "attn": dict(q=4 * 28 * 256, k=8 * 4 * 16 * 256, v=8 * 4 * 16 * 256, table=16, cu=8, lens=4, out=4 * 28 * 256,
                 lse=4 * 28 * 4, ws=2 * 148 * 256 * (128 * 4 + 8)),
}
CALLS = {"update": (update, UPDATE, {"past", "new"}), "append": (append, APPEND, {"qkv", "pos", "slots", "cos", "sin"}),
         "attn": (attn, ATTN, {"q", "k", "v", "table", "cu", "lens"})}


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no call can launch")
@pytest.mark.parametrize("name", CALLS)
def test_overlapping_arrays_are_refused(name):
    call, at, read = CALLS[name]
    assert call(**at) in (3, 4)  # past the checks: no device here
    for a in at:
        for b in at:
            if a == b:
                continue
            for shift in (0, SIZES[name][b] - 1 & ~31):  # b's first bytes, and its last ones
                got = call(**{**at, a: at[b] + shift})
                assert got == 1 if not {a, b} <= read else got in (3, 4), (a, b, shift)
            if b != "ws":  # right behind b
                assert call(**{**at, a: at[b] + (SIZES[name][b] + 31 & ~31)}) in (3, 4), (a, b)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no call can launch")
def test_one_row_may_be_rotated_in_place():
    assert append(**{**APPEND, "q": APPEND["qkv"], "T": 1}) in (3, 4)
    assert append(**{**APPEND, "q": APPEND["qkv"] + 256, "T": 1}) == 1


@pytest.mark.parametrize("call,args,bad", [
    (update, UPDATE, dict(B=0)), (update, UPDATE, dict(page=24)), (update, UPDATE, dict(tokens=-1)),
    (update, UPDATE, dict(table=None)), (update, UPDATE, dict(slots=None)), (update, UPDATE, dict(pages=1 << 28)),
    (append, APPEND, dict(D=80)), (append, APPEND, dict(max_pos=0)), (append, APPEND, dict(q=None)),
    (append, APPEND, dict(qkv=APPEND["qkv"] + 2)), (append, APPEND, dict(pages=1 << 28)),
    (attn, ATTN, dict(D=96)), (attn, ATTN, dict(scale=0.0)), (attn, ATTN, dict(out=ATTN["out"] + 4)),
    (attn, ATTN, dict(Hq=30)), (attn, ATTN, dict(page=48)), (attn, ATTN, dict(cu=None))])
def test_refusals_with_arrays_apart(call, args, bad):
    assert call(**{**args, **bad}) == 1
