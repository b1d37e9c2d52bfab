"""GPU: edges of the paged K/V cache operators: maxima that rise inside an item's
last block, captured loop bodies, empty steps, infinite scores, idle requests, long
prompts.  Tolerances as derived in test_paged_gpu."""
import ctypes
import math

import pytest
import torch

from test_paged_gpu import BF, FP, Paged, _i32, _no_device_error

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from std_b200 import ops as _ops

    assert torch.cuda.is_available()
    return _ops


def set_keys(x, b, keys):
    """Request b's keys of a Paged become `keys` [L, Hkv, D]."""
    x.keys[b] = (keys, x.keys[b][1])
    for i in range(-(-x.kv[b] // x.page)):
        rows = slice(i * x.page, min(x.kv[b], (i + 1) * x.page))
        x.k[x.table[b, i].item(), :, :rows.stop - rows.start] = keys[rows].permute(1, 0, 2)


# ------------------------------------------------------------------ running maxima
@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF)])
@pytest.mark.parametrize("tail", [0, 1, 15, 64, 65, 80, 127])
def test_maximum_rises_in_every_half_block(ops, D, dtype, tail):
    """Scores that jump by more than 2^8 from each 64 keys to the next, the last ones of
    an item included: O is rescaled in every half of every block, behind which no
    next score stands at an item's end.  Items of all forms follow one another in a CTA."""
    pairs = [(256 + tail, 1), (128 + tail, 19), (300 + tail, 3), (tail, 36), (512 + tail, 72), (700 + tail, 40)]
    pairs = pairs * 8 + [(2000 + tail, 25)] * 3
    x = Paged(pairs, 14, 2, D, 64, dtype, seed=tail)
    x.q = x.q.abs().clamp(0.5, 2)
    for b, (past, n) in enumerate(pairs):
        L = x.kv[b]
        half = torch.arange(L, device="cuda")[:, None, None] // 64
        set_keys(x, b, ((half + 1) * x.keys[b][0].float().abs().clamp(0.8, 1.2)).to(dtype))
    lse = torch.empty(x.q.shape[:2], device="cuda")
    for causal in (True, False):
        out = x.call(ops, causal, lse=lse)
        x.check(out, lse, causal)
        assert torch.equal(x.call(ops, causal), out)
    _no_device_error(ops)


# ------------------------------------------------------------------ workspaces and captured bodies
def test_workspace_of_the_caller(ops):
    """The same bits with a workspace kept over calls of different shapes; what is too
    small, misaligned or of another type is refused."""
    calls = [Paged([(4000, 1), (3000, 3)], 28, 4, 128, 16, BF, seed=1), Paged([(100, 900)], 8, 8, 128, 32, FP, seed=2),
             Paged([(9000, 1)], 28, 4, 128, 64, BF, seed=3)]
    ws = ops.paged_attention_workspace(128)
    for x in calls + calls:
        assert torch.equal(x.call(ops, workspace=ws), x.call(ops))
    x = calls[0]
    with pytest.raises(ValueError, match="workspace"):
        x.call(ops, workspace=ws[:-1])
    with pytest.raises(ValueError, match="workspace"):
        x.call(ops, workspace=torch.empty(ws.numel() + 16, dtype=torch.uint8, device="cuda")[16:])
    with pytest.raises(RuntimeError, match="workspace"):
        x.call(ops, workspace=ws.view(torch.int32))
    with pytest.raises(RuntimeError, match="workspace"):
        x.call(ops, workspace=ws.cpu())
    with pytest.raises(ValueError, match="head dim"):
        ops.paged_attention_workspace(96)
    _no_device_error(ops)


def _loop(body, done, count, limit):
    """`body` as the loop body of a graph being captured, run until done is set."""
    from std_b200 import _lib

    inner, h = _lib.capture_stream("while_body"), ctypes.c_ulonglong(0)
    _lib.call("std_capture_while_begin", torch.cuda.current_stream().cuda_stream, inner.cuda_stream, done.data_ptr(),
              done.numel(), count.data_ptr(), ctypes.byref(h), None)
    with torch.cuda.stream(inner):
        body()
    _lib.call("std_capture_while_end", inner.cuda_stream, h.value, done.data_ptr(), done.numel(), count.data_ptr(), limit)


def test_captured_loop_bodies(ops):
    """A loop body captures the calls with buffers of the caller's; its replays touch no
    memory that was given to others since.  Without them it refuses, as they would
    come from memory that does not stay with the graph."""
    a, b = Paged([(9000, 1), (40, 30)], 28, 4, 128, 16, BF, seed=1), Paged([(7000, 2), (50, 300)], 28, 4, 128, 64, BF, seed=2)
    want = [a.call(ops), b.call(ops)]
    done, graphs, kept = _i32([0]), [], []
    for x in (a, b):
        out, ws, count = torch.zeros_like(x.q), ops.paged_attention_workspace(128), _i32([0])
        lens = [n for _, n in x.pairs]
        past, new, held, n_free = _i32([p for p, _ in x.pairs]), _i32(lens), _i32([0] * 2), _i32([1000])
        table, free = torch.full((2, 800), -1, dtype=torch.int32, device="cuda"), torch.arange(1000, device="cuda").int()
        steps = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3, 2, sum(lens), sum(lens), 2)]

        def body():
            ops.paged_update(past, new, table, held, free, n_free, 16, sum(lens), out=steps)
            x.call(ops, out=out, workspace=ws)
            for kw in (dict(), dict(out=out), dict(workspace=ws)):
                with pytest.raises(RuntimeError, match="workspace="):
                    x.call(ops, **kw)
            with pytest.raises(RuntimeError, match="out="):
                ops.paged_update(past, new, table, held, free, n_free, 16, sum(lens))

        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            _loop(body, done, count, 3)
        graphs.append(g)
        kept.append((out, ws, count, steps, x.kv_lens, x.cu, past, new, table, held, free, n_free))
    torch.cuda.empty_cache()
    others = [torch.full((24 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(12)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for out, *_ in kept:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):  # both loops at once
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (out, _, count, steps, kv, cu, *_), w in zip(kept, want):
            assert torch.equal(out, w) and count.item() == 3
            assert torch.equal(steps[0], cu) and torch.equal(steps[1], kv)
        assert all((o == 7).all() for o in others)
    _no_device_error(ops)


def test_graphs_of_torch_need_no_workspace(ops):
    """Under torch.cuda.graph a call's own memory stays with the graph."""
    x = Paged([(9000, 1), (40, 300)], 28, 4, 128, 16, BF, seed=1)
    want, g = x.call(ops), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = x.call(ops)
    torch.cuda.empty_cache()
    others = [torch.full((24 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(6)]
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, want) and all((o == 7).all() for o in others)
    _no_device_error(ops)


# ------------------------------------------------------------------ scores of -inf
def far_below(x, lowest):
    """Every score of x strongly negative, and -inf at the keys `lowest(L)` (a mask)."""
    x.q = x.q.abs().clamp(0.5, 2)
    for b in range(len(x.pairs)):
        keys = (-40 * x.keys[b][0].float().abs().clamp(0.8, 1.2)).to(x.dtype)
        keys[lowest(x.kv[b])] = -math.inf
        set_keys(x, b, keys)


def check_hidden(x, out, lse, causal):
    """Paged.check for keys that hold -inf: such a key counts as hidden."""
    e, at, (Hq, D) = torch.finfo(x.dtype).eps, 0, x.q.shape[1:]
    G = Hq // x.k.shape[1]
    for b, (_, n) in enumerate(x.pairs):
        L = x.kv[b]
        q = x.q[at:at + n].double().permute(1, 0, 2)
        k, v = (t.double().permute(1, 0, 2).repeat_interleave(G, 0) for t in x.keys[b])
        hidden = k.isinf().any(-1)[:, None, :].expand(Hq, n, L)
        k = torch.where(k.isinf(), 0.0, k)
        if causal:
            hidden = hidden | (torch.arange(L, device="cuda")[None] > (L - n + torch.arange(n, device="cuda"))[:, None])
        s = (q @ k.transpose(1, 2) / math.sqrt(D)).masked_fill(hidden, -math.inf)
        size = (q.abs() @ k.abs().transpose(1, 2) / math.sqrt(D)).amax(-1, keepdim=True)
        m = s.amax(-1, keepdim=True)
        some = m > -math.inf
        p = torch.exp(s - torch.where(some, m, 0.0))
        l = torch.where(some, p.sum(-1, keepdim=True), 1.0)
        ref, A = p @ v / l, p @ v.abs() / l
        d = D * 2.0 ** -24 * size + 2.0 ** -22 + (34 + L / 64) * 2.0 ** -24
        tol = 1.01 * (e / 2 * ref.abs() + (e / 2 + 2 * d) * A)
        if x.dtype == FP:
            tol = tol + 2.0 ** -25 * (~hidden).double() @ v.abs() / l + 2.0 ** -25
        got = out[at:at + n].double().permute(1, 0, 2)
        assert torch.isfinite(got).all() and ((got - ref).abs() <= tol + 1e-30).all(), b
        want, g2 = torch.where(some, m + l.log(), -math.inf)[..., 0], lse[at:at + n].double().t()
        assert torch.equal(g2 == -math.inf, want == -math.inf), b
        fin = want > -math.inf
        t2 = 2 * d[..., 0] + (2 * want.abs() + 16) * 2.0 ** -22
        assert ((g2 - want).abs()[fin] <= t2[fin]).all(), b
        at += n


@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF)])
@pytest.mark.parametrize("first,count", [(0, 128), (0, 129), (0, 256), (0, 700), (128, 128), (64, 5000), (0, 100000)])
def test_scores_of_minus_infinity(ops, D, dtype, first, count):
    """Keys with a score of -inf over whole blocks, a request's first ones or all of them
    among these, before finite scores far below 0: they count as hidden, in every form
    (few rows, one tile, a pair, divided over CTAs)."""
    x = Paged([(300, 1), (290, 4), (290, 15), (200, 100), (1300, 2), (6000, 2), (3000, 30), (255, 1)], 14, 2, D, 64, dtype,
              seed=count)
    far_below(x, lambda L: (torch.arange(L, device="cuda") >= first) & (torch.arange(L, device="cuda") < first + count))
    lse = torch.empty(x.q.shape[:2], device="cuda")
    for causal in (True, False):
        out = x.call(ops, causal, lse=lse)
        check_hidden(x, out, lse, causal)
    _no_device_error(ops)


@pytest.mark.parametrize("new,D,dtype", [(1, 64, FP), (4, 128, BF), (12, 64, BF), (36, 128, FP)])
def test_scores_of_minus_infinity_past_the_long_sums(ops, new, D, dtype):
    """150 requests of 2^18 keys on the same pages, the first 153,600 keys with a score of
    -inf: a CTA's sums are put aside (after 2^17 keys at the latest) before any score counts."""
    L, page, G, B, start = 1 << 18, 256, 7, 150, 600
    g = torch.Generator(device="cuda").manual_seed(new)
    k = -40 * torch.randn(3, 1, page, D, generator=g, device="cuda").abs().clamp(0.8, 1.2)
    k[0, ..., 0] = -math.inf
    k = k.to(dtype)
    v = (torch.rand(3, 1, page, D, generator=g, device="cuda") + 0.5).to(dtype)
    ids = torch.arange(L // page, device="cuda")
    row = torch.where(ids < start, 0, 1 + ids % 2).int()
    q = torch.randn(B * new, G, D, generator=g, device="cuda").abs().clamp(0.5, 2).to(dtype)
    lse = torch.empty(B * new, G, device="cuda")
    cu, kv = torch.arange(0, B * new + 1, new, device="cuda").int(), torch.full((B,), L, device="cuda").int()
    out = ops.paged_attention(q, k, v, row.expand(B, -1).contiguous(), cu, kv, causal=False, lse=lse).double()
    s = torch.einsum("nhd,pkd->nhpk", q.double(), k[1:, 0].double()) / math.sqrt(D)
    size = torch.einsum("nhd,pkd->nhpk", q.double(), k[1:, 0].double().abs()).amax((-1, -2)) / math.sqrt(D)
    m = s.amax((-1, -2), keepdim=True)
    w = torch.exp(s - m) * ((L // page - start) / 2)
    l = w.sum((-1, -2))
    ref = torch.einsum("nhpk,pkd->nhd", w, v[1:, 0].double()) / l[..., None]
    e = torch.finfo(dtype).eps
    # output and probabilities rounded once each (v > 0: A = ref), scores as sums of D products, and sums of at
    # most 2^18 / 16 additions that are cut off (2^-23 of the sum each) in the products, 2^18 / 256 in l
    d = 2 * (D * 2.0 ** -24 * size + 2.0 ** -22)
    low = 2.0 ** -25 * (L - start * page) * v.max().double() / l if dtype == FP else torch.zeros_like(l)
    tol = (e + (2 ** 13 + 2 ** 9) * 2.0 ** -23 + d[..., None]) * ref + low[..., None]
    assert ((out - ref).abs() <= 1.01 * tol).all(), ((out - ref).abs() / tol).max().item()
    want = l.log() + m[..., 0, 0]
    assert ((lse.double() - want).abs() <= d + 2.0 ** 9 * 2.0 ** -23 + (2 * want.abs() + 16) * 2.0 ** -22).all()
    _no_device_error(ops)


@pytest.mark.parametrize("new,D,dtype", [(1, 64, FP), (4, 128, FP), (12, 64, FP), (36, 64, FP), (1, 64, BF), (36, 128, BF)])
@pytest.mark.parametrize("below", [19.3, 25.3])
def test_many_small_weights_beside_a_large_one(ops, new, D, dtype, below):
    """A first key that holds nearly all of a row and 2^17 others of 2^-below of its weight
    each, in one CTA (150 requests on the same pages).

    Half precision rounds such a probability to a multiple of 2^-24 of the kernel's unit,
    in which the largest is at least 2^7: off by at most 2^-32 of the largest weight.
    bf16 has the usual e / 2.  The sums: at most 2^17 / 16 additions that are cut off,
    2^-23 of the sum each."""
    L, page, G, B = 1 << 17, 256, 7, 150
    g = torch.Generator(device="cuda").manual_seed(new)
    k = torch.zeros(3, 1, page, D, device="cuda")
    k[..., 1] = 0.2 * torch.rand(3, 1, page, generator=g, device="cuda")
    k[0, 0, 0, 0] = below * math.log(2) * math.sqrt(D) / 4
    k = k.to(dtype)
    v = (torch.rand(3, 1, page, D, generator=g, device="cuda") + 0.5).to(dtype)
    v[0, 0, 0] = 0
    row = torch.arange(L // page, device="cuda").int() % 2 + 1
    row[0] = 0
    q = torch.zeros(B * new, G, D, device="cuda")
    q[..., 0] = 4
    q[..., 1] = torch.rand(B * new, G, generator=g, device="cuda")
    q = q.to(dtype)
    lse = torch.empty(B * new, G, device="cuda")
    cu, kv = torch.arange(0, B * new + 1, new, device="cuda").int(), torch.full((B,), L, device="cuda").int()
    out = ops.paged_attention(q, k, v, row.expand(B, -1).contiguous(), cu, kv, causal=False, lse=lse).double()
    count = torch.stack([(row == i).sum() for i in range(3)]).double()[:, None]
    s = torch.einsum("nhd,pkd->nhpk", q.double(), k[:, 0].double()) / math.sqrt(D)
    m = s.amax((-1, -2), keepdim=True)
    w = torch.exp(s - m) * count
    l = w.sum((-1, -2))
    ref = torch.einsum("nhpk,pkd->nhd", w, v[:, 0].double()) / l[..., None]
    e = torch.finfo(dtype).eps
    d = 2 * (D * 2.0 ** -24 * m[..., 0, 0].abs() + 2.0 ** -22)[..., None]
    tol = (e + 2.0 ** 13 * 2.0 ** -23 + d) * ref  # (v >= 0: the output's and the probabilities' e / 2)
    if dtype == FP:
        tol = tol + 2.0 ** -32 * L * v.max().double() + 2.0 ** -25
    assert ((out - ref).abs() <= 1.01 * tol).all(), ((out - ref).abs() / tol).max().item()
    want = l.log() + m[..., 0, 0]
    assert ((lse.double() - want).abs() <= d[..., 0] + 2.0 ** 9 * 2.0 ** -23 + (2 * want.abs() + 16) * 2.0 ** -22).all()
    _no_device_error(ops)


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("log2", [16, 20, 22, 23, 24, 25, 26, 27])
def test_scores_of_great_size(ops, dtype, log2):
    """Scores of 2^16 to 2^27, which 32 bits hold to 2^-8 to 8, with differences on both sides
    of what raises a maximum.  Their rounding decides the weights, so what holds is that
    each output is a mean of the values: between their least and greatest, but for the
    roundings of output and probabilities (e / 2 each, of one sign here) and the sums."""
    D, e = 128, torch.finfo(dtype).eps
    for step in (0.0, 4.0, 9.0, 14.0, 30.0):
        x = Paged([(700, 1), (690, 4), (2000, 15), (600, 100)], 14, 2, D, 64, dtype, seed=log2)
        big = 2 ** (log2 / 2) * math.sqrt(math.log(2) * math.sqrt(D))
        x.q = torch.zeros_like(x.q)
        x.q[..., 0], x.q[..., 1] = big, math.sqrt(D)
        x.keys = [(k, v.abs() + 0.5) for k, v in x.keys]
        x.v = x.v.abs() + 0.5
        for b in range(len(x.pairs)):
            keys, L = torch.zeros_like(x.keys[b][0]), x.kv[b]
            keys[..., 0] = big
            jump = torch.arange(L, device="cuda") // 64 % 5 * step
            keys[..., 1] = ((jump[:, None] + x.keys[b][0][..., 1].float()) * math.log(2)).to(dtype)
            set_keys(x, b, keys)
        lse = torch.empty(x.q.shape[:2], device="cuda")
        out, at = x.call(ops, lse=lse).double(), 0
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        for b, (_, n) in enumerate(x.pairs):
            v = x.keys[b][1].double().repeat_interleave(7, 1)
            lo, hi = v.amin(0), v.amax(0)
            slack = 1.01 * (e + 2.0 ** -12)
            assert (out[at:at + n] >= lo * (1 - slack)).all() and (out[at:at + n] <= hi * (1 + slack)).all(), (b, step)
            at += n
    _no_device_error(ops)


# ------------------------------------------------------------------ idle requests
@pytest.mark.parametrize("B", [33, 64, 2047, 8192])
def test_mostly_idle_batches(ops, B):
    """Requests without new tokens between those that have some, in runs of all lengths:
    the same rows as without them."""
    lens = {0: (700, 1), 1: (90, 20), B // 2: (40, 1), B - 33: (300, 3), B - 2: (1200, 2), B - 1: (64, 5)}
    lens = dict(sorted(lens.items()))  # (rows come in request order)
    x = Paged(list(lens.values()), 28, 4, 128, 16, BF, seed=B)
    x.check(x.call(ops), None)
    cu, kv, at = [0], [0] * B, dict(zip(lens, range(len(lens))))
    table = torch.full((B, x.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    for b in range(B):
        cu.append(cu[-1] + (lens[b][1] if b in lens else 0))
        if b in lens:
            kv[b], table[b] = sum(lens[b]), x.table[at[b]]
        elif b % 3 == 0:
            kv[b] = 50  # (keys, but no new tokens)
    out = ops.paged_attention(x.q, x.k, x.v, table, _i32(cu), _i32(kv))
    assert torch.equal(out, x.call(ops))
    _no_device_error(ops)


def test_idle_requests_are_passed_quickly(ops):
    """8192 requests, two at each end with a token: every CTA reads all lengths twice (about
    0.1 ms), whatever lies between its requests (passed one by one: 1.6 ms)."""
    from std_b200.timing import graph_time_us

    x = Paged([(999, 1)] * 4, 28, 4, 128, 64, BF)
    times = []
    for ids in ([0, 1, 2, 3], [0, 1, 8190, 8191]):
        new, kv = torch.zeros(8192, dtype=torch.int32), torch.zeros(8192, dtype=torch.int32)
        new[ids], kv[ids] = 1, 1000
        table = torch.full((8192, x.table.shape[1]), -1, dtype=torch.int32, device="cuda")
        table[ids] = x.table
        cu = torch.cat([torch.zeros(1), new.cumsum(0)]).int().cuda()
        kv, out = kv.cuda(), torch.empty_like(x.q)
        times.append(graph_time_us([lambda: ops.paged_attention(x.q, x.k, x.v, table, cu, kv, out=out)]))
        x.check(out, None)
    assert times[1] < 3 * times[0], times
    _no_device_error(ops)


# ------------------------------------------------------------------ tables
@pytest.mark.parametrize("max_tokens", [2 ** 31 - 256, 2 ** 31 - 1])
def test_update_with_the_most_tokens(ops, max_tokens):
    """Slots and positions for as many tokens as 32 bits count."""
    table, held = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), _i32([0, 0])
    free, n_free = torch.arange(8, dtype=torch.int32, device="cuda"), _i32([8])
    cu, kv, slots, pos, ok = ops.paged_update(_i32([3, 0]), _i32([20, 3]), table, held, free, n_free, 16, max_tokens)
    assert cu.tolist() == [0, 20, 23] and kv.tolist() == [23, 3] and ok.tolist() == [1, 1]
    assert slots[:23].tolist() == [7 * 16 + i for i in range(3, 16)] + [6 * 16 + i for i in range(7)] + [80, 81, 82]
    assert pos[:23].tolist() == list(range(3, 23)) + [0, 1, 2]
    assert slots.numel() == max_tokens and slots[23:].amax() == -1 and pos[23:].amax() == -1
    assert slots[23:].amin() == -1 and pos[23:].amin() == -1
    _no_device_error(ops)


def test_sizes_beyond_32_bits_are_refused(ops):
    """Sizes that differ from served ones by 2^32."""
    i = _i32([0])
    wide = torch.empty(1, 2 ** 32 + 8, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="page_size"):
        ops.paged_update(i, i, _i32([[-1] * 8]), i, i, i, 2 ** 32 + 16, 4)
    with pytest.raises(ValueError, match="max_blocks"):
        ops.paged_update(i, i, wide, i, i, i, 16, 4)
    with pytest.raises(ValueError, match="num_pages"):
        ops.paged_update(i, i, _i32([[-1] * 8]), i, wide.view(-1), i, 16, 4)
    x = Paged([(30, 2)], 28, 4, 128, 16, BF)
    with pytest.raises(ValueError, match="int32"):
        ops.paged_attention(x.q, x.k, x.v, wide, x.cu, x.kv_lens)
    _no_device_error(ops)


@pytest.mark.parametrize("graph", [False, True])
def test_steps_without_requests(ops, graph):
    """A server between requests: the three calls of a step with none, with rows for tokens
    and without."""
    cos = torch.ones(4, 64, dtype=BF, device="cuda")
    k = torch.full((5, 4, 16, 128), 3.0, dtype=BF, device="cuda")
    v = k.clone()
    for rows in (0, 6):
        qkv = torch.zeros(rows, 36 * 128, dtype=BF, device="cuda")
        q, out = (torch.full((rows, 28, 128), x, dtype=BF, device="cuda") for x in (4.0, 5.0))
        table, free, n_free = torch.empty(0, 7, dtype=torch.int32, device="cuda"), torch.arange(5, device="cuda").int(), _i32([5])
        none = _i32([])
        res = [torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (1, 0, rows, rows, 0)]

        def step(res):
            cu, kv, slots, pos, ok = ops.paged_update(none, none, table, none, free, n_free, 16, rows, out=res)
            ops.paged_rope_append(qkv, pos, slots, cos, cos, q, k, v)
            ops.paged_attention(q, k, v, table, cu, kv, out=out)
            return cu, kv, slots, pos, ok

        if graph:
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                got = step(res)
            g.replay()
        else:
            got = step(None)
        assert [t.tolist() for t in got] == [[0], [], [-1] * rows, [-1] * rows, []]
        assert (q == 4).all() and (out == 5).all() and (k == 3).all() and (v == 3).all() and n_free.item() == 5
        assert ops.paged_attention(q, k, v, table, got[0], none).shape == q.shape
    with pytest.raises(ValueError, match="page_size"):
        ops.paged_update(none, none, table, none, free, n_free, 24, 0)
    _no_device_error(ops)


def test_results_over_inputs_are_refused(ops):
    """Lengths advanced in place would lose a refused request's, q over qkv would race, out over
    a workspace or a pool too: refused, nothing changed.  One row may be rotated in place."""
    past, new, held, n_free = _i32([3, 0]), _i32([20, 3]), _i32([0, 0]), _i32([8])
    table, free = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.arange(8, device="cuda").int()
    e = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    for out in ((e(3), past, e(23), e(23), e(2)), (e(3), e(2), e(23), e(23), new), (e(3), held, e(23), e(23), e(2))):
        with pytest.raises(RuntimeError, match="status 1"):
            ops.paged_update(past, new, table, held, free, n_free, 16, 23, out=out)
    assert past.tolist() == [3, 0] and new.tolist() == [20, 3] and held.tolist() == [0, 0] and n_free.item() == 8
    cos = torch.ones(4, 64, dtype=BF, device="cuda")
    k = torch.zeros(5, 4, 16, 128, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.randn(3, 36 * 128, device="cuda").to(BF)
    before, i = qkv.clone(), _i32([0, 1, 2])
    with pytest.raises(RuntimeError, match="status 1"):
        ops.paged_rope_append(qkv, i, i, cos, cos, qkv.view(-1)[:3 * 28 * 128].view(3, 28, 128), k, v)
    with pytest.raises(RuntimeError, match="status 1"):
        ops.paged_rope_append(qkv, i, i, cos, cos, torch.empty(3, 28, 128, dtype=BF, device="cuda"), k, k)
    assert torch.equal(qkv, before) and (k == 0).all()
    one, sin = qkv[:1].clone(), torch.full_like(cos, 0.5)
    apart = ops.paged_rope_append(one, i[1:2], i[1:2], cos, sin, torch.empty(1, 28, 128, dtype=BF, device="cuda"), k, v)
    ops.paged_rope_append(one, i[1:2], i[1:2], cos, sin, one[:, :28 * 128].view(1, 28, 128), k, v)
    assert torch.equal(one[:, :28 * 128].view(1, 28, 128), apart)
    x = Paged([(30, 2)], 28, 4, 128, 16, BF)
    ws = ops.paged_attention_workspace(128)
    with pytest.raises(RuntimeError, match="status 1"):
        x.call(ops, workspace=ws, out=ws[:x.q.numel() * 2].view(BF).view(x.q.shape))
    with pytest.raises(RuntimeError, match="status 1"):
        x.call(ops, out=x.k.view(-1)[:x.q.numel()].view(x.q.shape))
    with pytest.raises(RuntimeError, match="status 1"):
        x.call(ops, lse=x.q.view(-1)[:x.q.shape[0] * 28 * 2].view(torch.float32).view(-1, 28))
    _no_device_error(ops)


# ------------------------------------------------------------------ long prompts
def test_long_prompt_every_row_against_64_bits(ops):
    """A 40,000-token prompt at once and in odd chunks: every row within its own rounding of
    the 64-bit value, e / 2 (|o| + A) with A = sum p |v| of that row.  The bound is sharp:
    each item (36 tokens of a key head's group) would miss it if its rows were zeros or
    those of the item before."""
    Hq, Hkv, D, page, n, item = 14, 2, 128, 128, 40000, 36
    G, e = Hq // Hkv, torch.finfo(BF).eps
    g = torch.Generator(device="cuda").manual_seed(2)
    blocks = -(-n // page)
    q = torch.randn(n, Hq, D, generator=g, device="cuda").to(BF)
    k = torch.randn(blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    v = torch.randn(blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    table = torch.randperm(blocks, generator=g, device="cuda").int().view(1, -1)
    whole = ops.paged_attention(q, k, v, table, _i32([0, n]), _i32([n]))
    parts, at = torch.empty_like(whole), 0
    for size in (1, 17, 5000, 13001, 36, 21944, 1):
        ops.paged_attention(q[at:at + size], k, v, table, _i32([0, size]), _i32([at + size]), out=parts[at:at + size])
        at += size
    assert at == n
    kk, vv = (t[table[0].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n].double() for t in (k, v))
    far = kk.norm(dim=-1).amax()
    before = None
    for a in range(0, n, 7 * item):
        b = min(n, a + 7 * item)
        hidden = torch.arange(b, device="cuda")[None] > torch.arange(a, b, device="cuda")[:, None]
        for h in range(Hkv):
            rows = q[a:b, h * G:(h + 1) * G].double()
            p = torch.einsum("thd,ld->htl", rows, kk[h, :b]).div_(math.sqrt(D)).masked_fill_(hidden, -math.inf)
            p = torch.softmax(p, -1)
            ref, A = torch.einsum("htl,ld->thd", p, vv[h, :b]), torch.einsum("htl,ld->thd", p, vv[h, :b].abs())
            del p
            # scores: sums of D products, |q| |k| at most; sums of n probabilities, 16 at a time and cut off (2^-23)
            d = D * 2.0 ** -24 * rows.norm(dim=-1, keepdim=True) * far / math.sqrt(D) + 2.0 ** -22 + (34 + n / 8) * 2.0 ** -24
            tol = 1.01 * (e / 2 * ref.abs() + (e / 2 + 2 * d) * A)
            for out in (whole, parts):
                off = (out[a:b, h * G:(h + 1) * G].double() - ref).abs()
                assert (off <= tol).all(), (a, h, (off / tol).max().item())
            others = torch.cat([ref[:item] if before is None else before, ref])[:b - a]
            before = ref[-item:] if h == Hkv - 1 else before
            for i in range(0, b - a, item):
                assert (ref[i:i + item].abs() > tol[i:i + item]).any(), (a, i, h)
                if a + i > 0:
                    assert ((others[i:i + item] - ref[i:i + item]).abs() > tol[i:i + item]).any(), (a, i, h)
    _no_device_error(ops)
