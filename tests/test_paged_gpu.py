"""GPU: the paged K/V cache operators (tables from lengths, append by slot,
attention over pages) against plain 64-bit implementations.

Tolerances.  e = finfo(dtype).eps; rounding to dtype is off by at most e / 2.
Attention: an output is rounded once (e/2 |o|) and each probability once (e/2,
so e/2 A with A = sum p |v| / sum p; half precision also loses up to 2^-25 of a
probability below 2^-14, the largest being at least 1 in the kernel's units).
Scores are 32-bit sums of D products: off by at most D 2^-24 sum |q k| scale each
way, which with the exponential's own 2^-22 is a relative error d of each
probability, in numerator and denominator: 2 d A.  Sums of n probabilities add
at most (34 + n / 64) 2^-24.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from std_b200 import ops as _ops

    assert torch.cuda.is_available()
    return _ops


def _no_device_error(ops):
    torch.cuda.synchronize()
    assert ops.device_error() == 0


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ attention
class Paged:
    """Random queries and a shuffled paged cache of requests with (past, new)
    lengths; everything no query may read is NaN."""

    def __init__(self, pairs, Hq, Hkv, D, page, dtype, seed=0, tail_rows=0, kv=None, spare=3, scale_q=1.5):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.pairs, self.page, self.dtype = pairs, page, dtype
        self.kv = [p + n for p, n in pairs] if kv is None else kv
        blocks = [-(-k // page) for k in self.kv]
        num_pages = sum(blocks) + spare
        ids = list(range(num_pages))
        rng.shuffle(ids)
        width = max(blocks + [1]) + 2
        table = torch.full((len(pairs), width), -1, dtype=torch.int32)
        k = torch.full((num_pages, Hkv, page, D), float("nan"))
        v = torch.full((num_pages, Hkv, page, D), float("nan"))
        self.keys, at = [], 0
        for b, nb in enumerate(blocks):
            mine = ids[at:at + nb]
            at += nb
            table[b, :nb] = torch.tensor(mine, dtype=torch.int32)
            L = self.kv[b]
            kb = torch.randn(L, Hkv, D, generator=g).to(dtype)
            vb = torch.randn(L, Hkv, D, generator=g).to(dtype)
            self.keys.append((kb.cuda(), vb.cuda()))
            for i, pg in enumerate(mine):
                rows = slice(i * page, min(L, (i + 1) * page))
                k[pg, :, :rows.stop - rows.start] = kb[rows].permute(1, 0, 2).float()
                v[pg, :, :rows.stop - rows.start] = vb[rows].permute(1, 0, 2).float()
        T = sum(n for _, n in pairs)
        self.q = (torch.randn(T + tail_rows, Hq, D, generator=g) * scale_q).to(dtype).cuda()
        self.k, self.v, self.table = k.to(dtype).cuda(), v.to(dtype).cuda(), table.cuda()
        cu = [0]
        for _, n in pairs:
            cu.append(cu[-1] + n)
        self.cu, self.kv_lens = _i32(cu), _i32(self.kv)

    def call(self, ops, causal=True, **kw):
        return ops.paged_attention(self.q, self.k, self.v, self.table, self.cu, self.kv_lens, causal=causal, **kw)

    def check(self, out, lse, causal=True, scale=None):
        Hq, D = self.q.shape[1:]
        scale = 1 / math.sqrt(D) if scale is None else scale
        e, at = torch.finfo(self.dtype).eps, 0
        for b, (_, n) in enumerate(self.pairs):
            L = self.kv[b]
            if n == 0:
                continue
            q = self.q[at:at + n].double().permute(1, 0, 2)                    # [Hq, n, D]
            G = Hq // self.k.shape[1]
            k = self.keys[b][0].double().permute(1, 0, 2).repeat_interleave(G, 0)
            v = self.keys[b][1].double().permute(1, 0, 2).repeat_interleave(G, 0)
            s = q @ k.transpose(1, 2) * scale
            size = (q.abs() @ k.abs().transpose(1, 2) * scale).amax(-1, keepdim=True) if L else s.new_zeros(Hq, n, 1)
            if causal:
                see = torch.arange(L, device="cuda")[None] <= (L - n + torch.arange(n, device="cuda"))[:, None]
                s = s.masked_fill(~see, -math.inf)
            m = s.amax(-1, keepdim=True) if L else s.new_full((Hq, n, 1), -math.inf)
            some = m > -math.inf
            p = torch.exp(s - torch.where(some, m, 0.0))
            l = p.sum(-1, keepdim=True)
            l1 = torch.where(some, l, 1.0)
            ref, A = p @ v / l1, p @ v.abs() / l1
            d = D * 2.0 ** -24 * size + 2.0 ** -22 + (34 + L / 64) * 2.0 ** -24
            tol = 1.01 * (e / 2 * ref.abs() + (e / 2 + 2 * d) * A)
            if self.dtype == torch.float16:
                tol = tol + 2.0 ** -25 * (see.double() if causal else torch.ones_like(s)) @ v.abs() / l1 + 2.0 ** -25
            got = out[at:at + n].double().permute(1, 0, 2)
            off = (got - ref).abs()
            assert torch.isfinite(got).all(), f"request {b}: non-finite output"
            assert (off <= tol + 1e-30).all(), f"request {b} (L {L}, n {n}): off by {(off - tol).max().item():.3e} over"
            if lse is not None:
                want = torch.where(some, torch.where(some, m, 0.0) + l1.log(), -math.inf)[..., 0]
                g2 = lse[at:at + n].double().t()
                assert torch.equal(g2 == -math.inf, want == -math.inf)
                fin = want > -math.inf
                t2 = 2 * d[..., 0] + (want.abs() + m[..., 0].abs() + 16) * 2.0 ** -22
                assert ((g2 - want).abs()[fin] <= t2[fin]).all()
            at += n


BF, FP = torch.bfloat16, torch.float16
CASES = [
    # pairs (past, new), Hq, Hkv, D, page, dtype, causal
    ([(0, 1)], 28, 4, 128, 16, BF, True),
    ([(199, 1)], 28, 4, 128, 16, BF, True),
    ([(126, 1), (127, 1), (128, 1), (255, 1), (256, 1)], 28, 4, 128, 64, BF, True),
    ([(300, 10), (1, 10), (1000, 18), (0, 18)], 28, 4, 128, 32, BF, True),
    ([(50, 19), (77, 36), (130, 37), (5, 73)], 7, 1, 128, 128, BF, True),
    ([(0, 0), (40, 3), (0, 0), (513, 0), (7, 1)], 28, 4, 128, 16, BF, True),
    ([(0, 500)], 28, 4, 128, 64, BF, True),
    ([(333, 301), (0, 129), (64, 1)], 16, 16, 64, 32, FP, True),
    ([(333, 301), (0, 129), (64, 1)], 16, 16, 64, 256, BF, False),
    ([(2000, 200), (90, 7)], 32, 8, 128, 256, FP, False),
    ([(700, 5), (3, 4)], 128, 1, 64, 16, BF, True),
    ([(700, 3), (3, 4), (1, 1)], 96, 2, 128, 32, FP, True),
    ([(3999, 1)], 28, 4, 128, 64, BF, True),
    ([(9000, 1), (20, 1)], 8, 1, 128, 16, BF, True),
    ([(6000, 40)], 12, 2, 128, 64, BF, True),
    ([(5, 1300)], 40, 8, 64, 16, FP, True),
    # rows of an item on both sides of 16, 32, 64 and 128, alone and beside each other
    ([(700, 2), (90, 3), (1300, 4), (2, 5), (640, 9), (31, 10), (128, 18), (0, 1)], 28, 4, 128, 64, BF, True),
    ([(2600, 1), (3, 2), (2000, 3), (900, 4), (77, 8)], 16, 1, 64, 16, FP, False),
    ([(1500, 32), (20, 33), (1, 16), (600, 64), (130, 17), (9, 128)], 4, 4, 128, 32, FP, True),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_against_64_bits(ops, case):
    pairs, Hq, Hkv, D, page, dtype, causal = CASES[case]
    x = Paged(pairs, Hq, Hkv, D, page, dtype, seed=case, tail_rows=3)
    T = x.q.shape[0]
    out = torch.full_like(x.q, 7.0)
    lse = torch.full((T, Hq), 7.0, device="cuda")
    got = x.call(ops, causal, out=out, lse=lse)
    assert got is out
    x.check(out, lse, causal)
    # rows behind the last request are left as they were
    assert (out[T - 3:] == 7).all() and (lse[T - 3:] == 7).all()
    # same inputs, same bits, with and without the log-sum-exp
    assert torch.equal(x.call(ops, causal)[:T - 3], out[:T - 3])
    _no_device_error(ops)


@pytest.mark.parametrize("B", [383, 385, 1000])
def test_attention_many_requests(ops, B):
    rng = random.Random(B)
    pairs = [(rng.randint(0, 60), rng.choice([0, 1, 1, 2, 20])) for _ in range(B)]
    x = Paged(pairs, 7, 1, 128, 16, BF, seed=B)
    x.check(x.call(ops), None)
    _no_device_error(ops)


def test_rows_without_keys(ops):
    """No keys at all, and fewer keys than new tokens: such rows give 0 and -inf."""
    x = Paged([(0, 4), (0, 20), (0, 40), (10, 2)], 28, 4, 128, 16, BF, kv=[0, 13, 1, 12])
    lse = torch.zeros(x.q.shape[:2], device="cuda")
    out = x.call(ops, lse=lse)
    x.check(out, lse)
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all()
    x.check(x.call(ops, causal=False), None, causal=False)
    _no_device_error(ops)


def test_large_scores_and_scale(ops):
    """Running maxima that jump (the accumulators are rescaled) and a user's scale."""
    for scale_q, scale in ((40.0, None), (3.0, 0.7), (1.0, 1e-3)):
        x = Paged([(1500, 30), (800, 1), (0, 300)], 28, 4, 128, 16, BF, seed=3, scale_q=scale_q)
        x.check(x.call(ops, scale=scale), None, scale=scale)
    _no_device_error(ops)


# ------------------------------------------------------------------ tables
def plain_update(past, new, table, n_blocks, free, n_free, page):
    """The rules of paged_update, one page at a time; changes table, n_blocks,
    free (a list) and returns the results and the new list length."""
    B, width = len(past), len(table[0])
    bad = [p < 0 or n < 0 or p + n > width * page or not 0 <= h <= width for p, n, h in zip(past, new, n_blocks)]
    want = [h if x else -(-(p + n) // page) for p, n, h, x in zip(past, new, n_blocks, bad)]
    back = [(b, j) for b in range(B) for j in range(want[b], n_blocks[b])]
    stack = free[:n_free] + [table[b][j] for b, j in reversed(back)]
    for b, j in back:
        table[b][j] = -1
    pool, ok, full = len(stack), [], False
    free[:pool] = stack
    for b in range(B):
        need = max(0, want[b] - n_blocks[b])
        full = full or need > pool
        ok.append(not bad[b] and (need == 0 or not full))
        if ok[b]:
            for j in range(n_blocks[b], want[b]):
                pool -= 1
                table[b][j] = free[pool]
            n_blocks[b] = want[b]
    cu, slots, positions = [0], [], []
    for b in range(B):
        for x in range(past[b], past[b] + new[b]) if ok[b] else [None] * max(0, new[b]):
            positions.append(-1 if x is None else x)
            slots.append(-1 if x is None else table[b][x // page] * page + x % page)
        cu.append(cu[-1] + max(0, new[b]))
    kv = [p + n if o else 0 for p, n, o in zip(past, new, ok)]
    return cu, kv, slots, positions, [int(o) for o in ok], pool


class Tables:
    """The state on the device and beside it in lists."""

    def __init__(self, B, width, num_pages, page, seed):
        self.rng = random.Random(seed)
        ids = list(range(num_pages))
        self.rng.shuffle(ids)
        self.page, self.free, self.n_free = page, ids, num_pages
        self.table, self.n_blocks = [[-1] * width for _ in range(B)], [0] * B
        self.dev = [_i32(self.table), _i32(self.n_blocks), _i32(self.free), _i32([self.n_free])]

    def step(self, ops, past, new, max_tokens, stream_out=None):
        got = ops.paged_update(_i32(past), _i32(new), *self.dev, self.page, max_tokens, out=stream_out)
        cu, kv, slots, pos, ok, self.n_free = plain_update(past, new, self.table, self.n_blocks, self.free, self.n_free,
                                                           self.page)
        slots, pos = (slots + [-1] * max_tokens)[:max_tokens], (pos + [-1] * max_tokens)[:max_tokens]
        for g, w, name in zip(got, (cu, kv, slots, pos, ok), ("cu_q", "kv_lens", "slots", "positions", "admitted")):
            assert g.tolist() == w, name
        for g, w, name in zip(self.dev, (self.table, self.n_blocks, None, [self.n_free]),
                              ("block_table", "n_blocks", "", "n_free")):
            assert w is None or g.tolist() == w, name
        assert self.dev[2].tolist()[:self.n_free] == self.free[:self.n_free], "free_pages"
        return kv, ok


@pytest.mark.parametrize("B,width,pages,page,most", [(1, 4, 5, 16, 20), (8, 40, 200, 64, 30), (33, 12, 150, 32, 60),
                                                     (300, 20, 2500, 16, 40), (1500, 9, 4000, 128, 200)])
def test_update_random_steps(ops, B, width, pages, page, most):
    """A serving loop's steps: growth, rollback, release, refusals for lack of pages."""
    x = Tables(B, width, pages, page, seed=B)
    lens = [0] * B
    for step in range(6):
        new = [0 if x.rng.random() < 0.2 else x.rng.randint(0, most) for _ in range(B)]
        past = [min(p, width * page - n) if x.rng.random() < 0.9 else 0 for p, n in zip(lens, new)]
        total = sum(new)
        kv, ok = x.step(ops, past, new, max(0, total + x.rng.choice([0, 0, 5])))
        lens = [k if o else p for k, o, p in zip(kv, ok, past)]
        if step % 2:  # some of the new tokens are given up again
            lens = [max(0, p - x.rng.randint(0, most)) for p in lens]
            kv, ok = x.step(ops, lens, [0] * B, 0)
    _no_device_error(ops)


def test_update_take_then_return_restores_everything(ops):
    x = Tables(20, 30, 400, 16, seed=5)
    past = [x.rng.randint(0, 200) for _ in range(20)]
    x.step(ops, past, [0] * 20, 0)
    before = [t.clone() for t in x.dev]
    x.step(ops, past, [x.rng.randint(0, 100) for _ in range(20)], 2000)
    x.step(ops, past, [0] * 20, 0)
    for a, b in zip(before, x.dev):
        assert torch.equal(a, b)


def test_update_many_tokens(ops):
    """More tokens than one block's threads, odd counts, one request holding most."""
    x = Tables(9, 700, 3000, 16, seed=6)
    x.step(ops, [0, 100, 7, 0, 3, 0, 0, 1, 2], [9001, 1, 0, 0, 130, 77, 16, 15, 17], 9300)
    x.step(ops, [9001, 101, 7, 0, 133, 77, 16, 16, 19], [1200] + [600] * 8, 1200 + 600 * 8)
    _no_device_error(ops)


def test_update_reports_bad_lengths(ops):
    """A negative length or one past the table refuses that request alone; too
    many tokens and bad page ids are reported and nothing is written past the
    outputs."""
    x = Tables(4, 4, 30, 16, seed=7)
    x.step(ops, [0, -5, 60, 3], [10, 4, 10, 2], 40)
    assert ops.device_error() == 3
    x.step(ops, [10, 0, 0, 5], [3, 0, 2, -1], 40)
    assert ops.device_error() == 3
    outs = [torch.full((n,), 99, dtype=torch.int32, device="cuda") for n in (5, 4, 8, 8, 4)]
    guard = torch.full((3, 8), 99, dtype=torch.int32, device="cuda")
    ops.paged_update(_i32([13, 0, 2, 5]), _i32([20, 0, 0, 0]), *x.dev, 16, 8, out=(outs[0], outs[1], guard[0], guard[1], outs[4]))
    assert (guard[2] == 99).all() and guard[1].tolist() == list(range(13, 21))
    assert ops.device_error() == 3
    table = _i32([[1000, -1]])
    got = ops.paged_update(_i32([4]), _i32([2]), table, _i32([1]), _i32([0, 1]), _i32([0]), 16, 2)
    assert got[2].tolist() == [-1, -1] and ops.device_error() == 2
    got = ops.paged_update(_i32([0]), _i32([2]), _i32([[-1, -1]]), _i32([0]), _i32([3, 1]), _i32([50]), 16, 2)
    assert got[2].tolist() == [16, 17] and ops.device_error() == 2  # the list cut to its two entries
    _no_device_error(ops)


# ------------------------------------------------------------------ append
def _rope_tables(n, D, dtype):
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv[None]
    return a.cos().to(dtype).cuda(), a.sin().to(dtype).cuda()


@pytest.mark.parametrize("T,Hq,Hkv,D,page,dtype", [(1, 28, 4, 128, 16, BF), (80, 28, 4, 128, 64, BF),
                                                    (333, 7, 1, 128, 256, FP), (1001, 16, 16, 64, 32, FP),
                                                    (17, 40, 8, 64, 128, BF), (5, 96, 32, 128, 16, BF)])
def test_append(ops, T, Hq, Hkv, D, page, dtype):
    g = torch.Generator().manual_seed(T)
    num_pages, max_pos = -(-T // page) + 4, 5000
    cos, sin = _rope_tables(max_pos, D, dtype)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(dtype).cuda()
    pos = torch.randint(0, max_pos, (T,), generator=g).int()
    slots = torch.randperm(num_pages * page, generator=g)[:T].int()
    if T > 4:
        pos[2], slots[2] = -1, -1      # no token here
        slots[4] = -1                  # rotated, not stored
    k = torch.full((num_pages, Hkv, page, D), 5.0, dtype=dtype, device="cuda")
    v, q = torch.full_like(k, 6.0), torch.full((T, Hq, D), 4.0, dtype=dtype, device="cuda")
    assert ops.paged_rope_append(qkv, pos.cuda(), slots.cuda(), cos, sin, q, k, v) is q
    x = qkv.double().view(T, -1, D)
    c, s = cos.double()[pos.clamp(min=0).cuda().long()][:, None], sin.double()[pos.clamp(min=0).cuda().long()][:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    # one rounding to dtype after two products and a sum in 32 bits
    size = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
    tol = torch.finfo(dtype).eps / 2 * y.abs() * 1.001 + 3 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == FP else 0)
    have = (pos >= 0).cuda()
    assert ((q.double() - y[:, :Hq]).abs() <= tol[:, :Hq])[have].all()
    assert (q[~have] == 4).all()
    rows = k.permute(0, 2, 1, 3).reshape(-1, Hkv, D), v.permute(0, 2, 1, 3).reshape(-1, Hkv, D)
    kept = (slots >= 0).cuda()
    at = slots.cuda().long()[kept]
    assert ((rows[0][at].double() - y[kept][:, Hq:Hq + Hkv]).abs() <= tol[kept][:, Hq:Hq + Hkv]).all()
    assert torch.equal(rows[1][at], qkv.view(T, -1, D)[kept][:, Hq + Hkv:])
    other = torch.ones(num_pages * page, dtype=torch.bool, device="cuda")
    other[at] = False
    assert (rows[0][other] == 5).all() and (rows[1][other] == 6).all()
    _no_device_error(ops)


def test_append_reports_out_of_range(ops):
    cos, sin = _rope_tables(10, 64, BF)
    qkv = torch.randn(3, 3 * 64, device="cuda").to(BF)
    k = torch.zeros(2, 1, 16, 64, dtype=BF, device="cuda")
    v, q = torch.zeros_like(k), torch.zeros(3, 1, 64, dtype=BF, device="cuda")
    ops.paged_rope_append(qkv, _i32([0, 10, 2]), _i32([0, 1, 32]), cos, sin, q, k, v)
    assert ops.device_error() == 2
    assert torch.equal(v[0, 0, :2], qkv[:2, 128:]) and (v.view(-1, 64)[2:] == 0).all()
    last = torch.zeros_like(q)
    ops.paged_rope_append(qkv, _i32([0, 9, 2]), _i32([-1, -1, -1]), cos, sin, last, k, v)
    assert torch.equal(last[1], q[1])  # read as the last position
    _no_device_error(ops)


# ------------------------------------------------------------------ misuse, and odd use
def test_attention_bad_entries_are_reported(ops):
    """Page ids, lengths and token ranges that do not fit: reported, nothing read or
    written out of range, the other requests right."""
    x = Paged([(300, 4), (200, 30), (90, 1), (40, 50)], 28, 4, 128, 16, BF, seed=1)
    good = x.call(ops)
    x.check(good, None)
    for bad in (-7, x.k.shape[0], 2 ** 30):
        keep = x.table[0, 3].item()
        x.table[0, 3] = bad
        out = x.call(ops)
        assert ops.device_error() == 2
        assert torch.isfinite(out[:4]).all() and torch.equal(out[4:], good[4:])
        x.table[0, 3] = keep
    # (request 1 has 15 pages; a length cut to the table's width reaches the -1 behind them)
    room = x.table.shape[1] * 16
    table = torch.where(x.table < 0, 0, x.table)
    for lens in ([304, -3, 91, 90], [304, room + 1, 91, 90], [304, 2 ** 31 - 1, 91, 90]):
        out = torch.full_like(x.q, 3.0)
        ops.paged_attention(x.q, x.k, x.v, table, x.cu, _i32(lens), out=out)
        assert ops.device_error() == 3
        assert torch.equal(out[:4], good[:4]) and torch.equal(out[34:35], good[34:35])
    for cu in ([0, 4, 34, 35, 86], [0, 4, 2, 35, 85], [0, -4, 34, 35, 85], [-1, 4, 34, 35, 85]):
        out = torch.full_like(x.q, 3.0)
        ops.paged_attention(x.q, x.k, x.v, x.table, _i32(cu), x.kv_lens, out=out)
        assert ops.device_error() == 3
    out = torch.full_like(x.q, 3.0)
    ops.paged_attention(x.q, x.k, x.v, x.table, _i32([0, 4, 34, 35, 86]), x.kv_lens, out=out)
    assert ops.device_error() == 3
    assert torch.equal(out[:35], good[:35]) and (out[35:] == 3).all()  # the last request skipped
    _no_device_error(ops)


def test_attention_no_tokens(ops):
    x = Paged([(30, 0), (5, 0)], 28, 4, 128, 16, BF, tail_rows=4)
    out = torch.full_like(x.q, 3.0)
    x.call(ops, out=out)
    assert (out == 3).all()
    none = x.q[:0]
    assert ops.paged_attention(none, x.k, x.v, x.table, x.cu, x.kv_lens).shape == (0, 28, 128)
    _no_device_error(ops)


def test_attention_shared_pages_and_order(ops):
    """Requests that share their first pages, and the same request in other batches
    and places: within rounding of one another."""
    x = Paged([(1000, 3), (700, 40), (64, 1)], 28, 4, 128, 32, BF, seed=2)
    out = x.call(ops)
    x.check(out, None)
    table = torch.stack([x.table[1], x.table[0], x.table[1]])
    q = torch.cat([x.q[3:43], x.q[:3], x.q[3:43]])
    o2 = ops.paged_attention(q, x.k, x.v, table, _i32([0, 40, 43, 83]), _i32([740, 1003, 740]))
    x2 = Paged.__new__(Paged)
    x2.__dict__.update(x.__dict__, pairs=[(700, 40), (1000, 3), (700, 40)], kv=[740, 1003, 740], q=q,
                       keys=[x.keys[1], x.keys[0], x.keys[1]])
    x2.check(o2, None)
    _no_device_error(ops)


def test_attention_offsets_beyond_32_bits(ops):
    """Pools of more than 2^32 bytes and 2^31 elements, the pages used at their end and
    their start."""
    num_pages, Hkv, page, D = 70000, 4, 64, 128  # 2.3e9 elements a pool
    k = torch.empty(num_pages, Hkv, page, D, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    small = Paged([(500, 3), (100, 40)], 28, Hkv, D, page, BF, seed=8)
    ids = [num_pages - 1 - 3 * i if i % 2 == 0 else i for i in range(small.k.shape[0])]
    k[ids], v[ids] = small.k, small.v
    table = torch.where(small.table >= 0, torch.tensor(ids, dtype=torch.int32, device="cuda")[small.table.clamp(min=0).long()],
                        -1)
    out = ops.paged_attention(small.q, k, v, table.int().contiguous(), small.cu, small.kv_lens)
    assert torch.equal(out, small.call(ops))
    cos, sin = _rope_tables(16, D, BF)
    qkv = torch.randn(2, (28 + 2 * Hkv) * D, device="cuda").to(BF)
    q = torch.empty(2, 28, D, dtype=BF, device="cuda")
    ops.paged_rope_append(qkv, _i32([0, 0]), _i32([num_pages * page - 1, 5]), cos, sin, q, k, v)
    want = qkv.view(2, -1, D)  # position 0: no rotation
    assert torch.equal(k[-1, :, -1], want[0, 28:32]) and torch.equal(v[-1, :, -1], want[0, 32:])
    assert torch.equal(k[0, :, 5], want[1, 28:32]) and torch.equal(q, want[:, :28])
    _no_device_error(ops)


def test_attention_scores_of_one_sign_and_infinities_behind_the_end(ops):
    """Strongly negative scores everywhere (exponentials far below the first guess of
    the maximum), and +-inf instead of NaN in the rows that no query may read."""
    for dtype in (BF, FP):
        x = Paged([(700, 1), (300, 50), (10, 9)], 8, 2, 128, 64, dtype, seed=4)
        x.q = x.q.abs()
        x.keys = [(-k.abs(), v) for k, v in x.keys]
        for b, (kb, _) in enumerate(x.keys):
            for i in range(-(-x.kv[b] // 64)):
                rows = slice(i * 64, min(x.kv[b], (i + 1) * 64))
                x.k[x.table[b, i].item(), :, :rows.stop - rows.start] = kb[rows].permute(1, 0, 2)
        x.k = torch.where(x.k.isnan(), float("inf"), x.k).to(dtype)
        x.v = torch.where(x.v.isnan(), float("-inf"), x.v).to(dtype)
        lse = torch.empty(x.q.shape[:2], device="cuda")
        x.check(x.call(ops, lse=lse), lse)
    _no_device_error(ops)


def test_two_streams_and_repeated_calls(ops):
    """Calls on two streams at once do not disturb one another."""
    a, b = Paged([(4000, 1), (3000, 3)], 28, 4, 128, 16, BF, seed=1), Paged([(100, 900)], 16, 16, 64, 32, FP, seed=2)
    want_a, want_b = a.call(ops), b.call(ops)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got_a, got_b = [], []
    for _ in range(8):
        with torch.cuda.stream(s1):
            got_a.append(a.call(ops))
        with torch.cuda.stream(s2):
            got_b.append(b.call(ops))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want_a) for g in got_a) and all(torch.equal(g, want_b) for g in got_b)
    _no_device_error(ops)


def test_wrapper_refusals(ops):
    x = Paged([(30, 2)], 28, 4, 128, 16, BF)
    with pytest.raises(RuntimeError, match="float32"):
        ops.paged_attention(x.q.float(), x.k, x.v, x.table, x.cu, x.kv_lens)
    with pytest.raises(RuntimeError, match="k_pages"):
        ops.paged_attention(x.q.half(), x.k, x.v, x.table, x.cu, x.kv_lens)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.paged_attention(x.q, x.k.transpose(1, 2).contiguous().transpose(1, 2), x.v, x.table, x.cu, x.kv_lens)
    with pytest.raises(ValueError, match="v_pages"):
        ops.paged_attention(x.q, x.k, x.v[:-1], x.table, x.cu, x.kv_lens)
    with pytest.raises(ValueError, match="cu_q"):
        ops.paged_attention(x.q, x.k, x.v, x.table, x.cu[:1], x.kv_lens)
    with pytest.raises(ValueError, match="multiple"):
        ops.paged_attention(x.q[:, :27].contiguous(), x.k, x.v, x.table, x.cu, x.kv_lens)
    with pytest.raises(ValueError, match="scale"):
        ops.paged_attention(x.q, x.k, x.v, x.table, x.cu, x.kv_lens, scale=0.0)
    with pytest.raises(ValueError, match="page_size"):
        ops.paged_attention(x.q, x.k[:, :, :8].contiguous(), x.v[:, :, :8].contiguous(), x.table, x.cu, x.kv_lens)
    with pytest.raises(RuntimeError, match="status 1"):
        ops.paged_attention(x.q, x.k, x.v, x.table, x.cu, x.kv_lens, out=x.q)
    with pytest.raises(RuntimeError, match="int32"):
        ops.paged_update(x.kv_lens.long(), x.kv_lens, x.table, x.kv_lens, x.kv_lens, x.kv_lens, 16, 4)
    with pytest.raises(ValueError, match="n_free"):
        ops.paged_update(x.kv_lens, x.kv_lens, x.table, x.kv_lens, x.kv_lens, x.cu, 16, 4)
    with pytest.raises(RuntimeError, match="status 1"):
        ops.paged_update(x.kv_lens, x.kv_lens, x.table, x.kv_lens, x.kv_lens, x.kv_lens, 24, 4)
    _no_device_error(ops)


# ------------------------------------------------------------------ together
def _serve(ops, graph):
    """A server's steps over one layer: prompts in chunks beside decoding requests,
    drafts given up again, requests that end and make room, one that has to wait."""
    Hq, Hkv, D, page, num_pages, width, B, rows = 28, 4, 128, 16, 40, 24, 4, 160
    g = torch.Generator().manual_seed(9)
    cos, sin = _rope_tables(width * page, D, BF)
    k = torch.full((num_pages, Hkv, page, D), float("nan"), dtype=BF, device="cuda")
    v = torch.full_like(k, float("nan"))
    ids = list(range(num_pages))
    random.Random(3).shuffle(ids)
    table, n_blocks = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), _i32([0] * B)
    free, n_free = _i32(ids), _i32([num_pages])
    past, new = _i32([0] * B), _i32([0] * B)
    qkv = torch.zeros(rows, (Hq + 2 * Hkv) * D, dtype=BF, device="cuda")
    q, out = torch.zeros(rows, Hq, D, dtype=BF, device="cuda"), torch.zeros(rows, Hq, D, dtype=BF, device="cuda")
    step_out = tuple(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (B + 1, B, rows, rows, B))

    def run():
        cu, kv_lens, slots, positions, _ = ops.paged_update(past, new, table, n_blocks, free, n_free, page, rows,
                                                            out=step_out)
        ops.paged_rope_append(qkv, positions, slots, cos, sin, q, k, v)
        ops.paged_attention(q, k, v, table, cu, kv_lens, out=out)

    run()  # nothing new: allocates and loads before the capture
    if graph:
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            run()
    hist = [[] for _ in range(B)]  # each request's (rotated k, v) so far
    e = torch.finfo(BF).eps
    #        past lengths, new tokens, which are admitted
    steps = [([0, 0, 0, 0], [100, 30, 7, 0], [1, 1, 1, 1]),
             ([100, 30, 7, 0], [1, 10, 120, 0], [1, 1, 1, 1]),
             ([101, 33, 127, 0], [1, 1, 1, 90], [1, 1, 1, 1]),        # 7 of 10 drafts given up
             ([102, 34, 128, 90], [60, 70, 1, 20], [1, 1, 1, 1]),
             ([162, 104, 129, 110], [100, 1, 1, 50], [1, 1, 1, 0]),   # the last one does not fit
             ([0, 105, 130, 110], [0, 1, 1, 50], [1, 1, 1, 1])]       # the first one has ended
    for past_l, new_l, admitted in steps:
        past.copy_(_i32(past_l))
        new.copy_(_i32(new_l))
        x = torch.randn(rows, (Hq + 2 * Hkv) * D, generator=g).to(BF)
        qkv.copy_(x)
        out.fill_(9.0)
        cg.replay() if graph else run()
        assert step_out[4].tolist() == admitted
        at = 0
        for b, (p, n) in enumerate(zip(past_l, new_l)):
            mine = x[at:at + n].view(n, Hq + 2 * Hkv, D).cuda()
            if not admitted[b]:
                assert (out[at:at + n] == 0).all()
                at += n
                continue
            pos = torch.arange(p, p + n, device="cuda")
            y = mine.double()
            lo, hi = y[..., :D // 2], y[..., D // 2:]
            c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
            y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(BF)
            hist[b] = hist[b][:p] + [(y[i, Hq:Hq + Hkv], mine[i, Hq + Hkv:]) for i in range(n)]
            at += n
            if n == 0:
                continue
            G = Hq // Hkv
            kb = torch.stack([h[0] for h in hist[b]]).double().permute(1, 0, 2).repeat_interleave(G, 0)
            vb = torch.stack([h[1] for h in hist[b]]).double().permute(1, 0, 2).repeat_interleave(G, 0)
            qb = y[:, :Hq].double().permute(1, 0, 2)
            s_ = qb @ kb.transpose(1, 2) / math.sqrt(D)
            size = (qb.abs() @ kb.abs().transpose(1, 2) / math.sqrt(D)).amax(-1, keepdim=True)
            see = torch.arange(p + n, device="cuda")[None] <= pos[:, None]
            pr = torch.softmax(s_.masked_fill(~see, -math.inf), -1)
            ref, A = pr @ vb, pr @ vb.abs()
            # on top of the attention's own rounding, a q or k rounded the other way (rope in 32 bits against
            # 64, ties aside) moves a score by at most e of its size
            d = e * size + D * 2.0 ** -24 * size + 2.0 ** -20
            tol = 1.01 * (e / 2 * ref.abs() + (e / 2 + 2 * d) * A)
            got = out[at - n:at].double().permute(1, 0, 2)
            assert ((got - ref).abs() <= tol).all(), (b, p, n)
        assert (out[at:] == 9).all()
    held = sum(n_blocks.tolist())
    assert held + n_free.item() == num_pages
    used = [i for b in range(B) for i in table[b].tolist() if i >= 0] + free[:n_free.item()].tolist()
    assert sorted(used) == list(range(num_pages))
    _no_device_error(ops)


def test_serving_steps(ops):
    _serve(ops, graph=False)


def test_serving_steps_from_a_graph(ops):
    """The same steps replayed from one captured graph: lengths, pages and splits are
    all found on the device."""
    _serve(ops, graph=True)


def test_two_graphs_at_once(ops):
    """Graphs captured one after the other share no workspace: replayed on two streams
    at the same time, both are right."""
    a, b = Paged([(9000, 1)], 28, 4, 128, 16, BF, seed=1), Paged([(7000, 2), (50, 3)], 28, 4, 128, 64, BF, seed=2)
    want = [a.call(ops), b.call(ops)]
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        out = torch.zeros_like(x.q)
        with torch.cuda.graph(g):
            x.call(ops, out=out)
        graphs.append(g)
        outs.append(out)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    _no_device_error(ops)


# ------------------------------------------------------------------ extremes
def test_attention_wide_tables(ops):
    """Tables that allow requests of 2^31 keys: costs are counted in coarser units,
    the shares stay a partition of the blocks."""
    x = Paged([(3000, 1), (700, 40), (0, 300), (5000, 2), (90, 1), (1, 1), (2000, 9), (12, 130)], 28, 4, 128, 256, BF,
              seed=6)
    wide = torch.full((8, 8388600), -1, dtype=torch.int32, device="cuda")
    wide[:, :x.table.shape[1]] = x.table
    out = torch.empty_like(x.q)
    lse = torch.empty(x.q.shape[:2], device="cuda")
    ops.paged_attention(x.q, x.k, x.v, wide, x.cu, x.kv_lens, out=out, lse=lse)
    x.check(out, lse)
    _no_device_error(ops)


@pytest.mark.parametrize("offset", [8, 16, 24])
def test_attention_tensors_inside_others(ops, offset):
    """Tensors that begin 16 bytes into an allocation (16-byte, not 32-byte aligned)."""
    x = Paged([(300, 1), (70, 60), (2500, 9)], 28, 4, 128, 64, BF, seed=offset)
    want = x.call(ops)

    def inside(t):
        room = torch.zeros(t.numel() + offset, dtype=t.dtype, device="cuda")
        view = room[offset:].view(t.shape)
        view.copy_(t)
        return view

    out = inside(torch.zeros_like(x.q))
    got = ops.paged_attention(inside(x.q), inside(x.k), inside(x.v), inside(x.table), inside(x.cu), inside(x.kv_lens),
                              out=out)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="status 1"):
        room = torch.zeros(x.q.numel() + 1, dtype=BF, device="cuda")
        ops.paged_attention(x.q, x.k, x.v, x.table, x.cu, x.kv_lens, out=room[1:].view(x.q.shape))
    _no_device_error(ops)


def test_attention_most_requests_and_many_heads(ops):
    rng = random.Random(8192)
    x = Paged([(rng.randint(0, 40), rng.choice([0, 1, 1, 2])) for _ in range(8192)], 2, 1, 64, 16, FP, seed=3)
    out = x.call(ops)
    for b in (0, 1, 4095, 8190, 8191):  # (the 64-bit check of all would take minutes)
        n = x.pairs[b][1]
        one = Paged.__new__(Paged)
        at = x.cu[b].item()
        one.__dict__.update(x.__dict__, pairs=[x.pairs[b]], kv=[x.kv[b]], keys=[x.keys[b]], q=x.q[at:at + n])
        one.check(out[at:at + n], None)
    assert torch.isfinite(out).all()
    x = Paged([(100, 3), (9, 1), (700, 140)], 300, 300, 64, 32, BF, seed=4)
    x.check(x.call(ops), None)
    _no_device_error(ops)


def test_long_prompt_whole_and_in_chunks(ops):
    """A 40,000-token prompt at once and in odd chunks: the same rows within their rounding."""
    Hq, Hkv, D, page, n = 14, 2, 128, 128, 40000
    g = torch.Generator(device="cuda").manual_seed(1)
    blocks = -(-n // page)
    q = torch.randn(n, Hq, D, generator=g, device="cuda").to(BF)
    k = torch.randn(blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    v = torch.randn(blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    table = torch.randperm(blocks, generator=g, device="cuda").int().view(1, -1)
    whole = ops.paged_attention(q, k, v, table, _i32([0, n]), _i32([n]))
    at = 0
    for size in (1, 17, 5000, 13001, 36, 21944, 1):
        part = ops.paged_attention(q[at:at + size], k, v, table, _i32([0, size]), _i32([at + size]))
        # each is off from the exact row by at most e/2 (|o| + A), A <= max |v| here taken as 6
        off = (part.double() - whole[at:at + size].double()).abs()
        assert (off <= 2 * 2.0 ** -8 * (whole[at:at + size].double().abs() + 6)).all()
        assert off.mean() < 1e-3
        at += size
    assert at == n
    # rows near the end against 64 bits
    kk = k[table[0].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n].double()
    vv = v[table[0].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n].double()
    for row in (n - 1, n - 129, 20000):
        s = torch.einsum("hd,hld->hl", q[row].double(), kk[:, :row + 1].repeat_interleave(7, 0)) / math.sqrt(D)
        p = torch.softmax(s, -1)
        ref = torch.einsum("hl,hld->hd", p, vv[:, :row + 1].repeat_interleave(7, 0))
        A = torch.einsum("hl,hld->hd", p, vv[:, :row + 1].abs().repeat_interleave(7, 0))
        assert ((whole[row].double() - ref).abs() <= 1.02 * 2.0 ** -8 * (ref.abs() + A)).all()
    _no_device_error(ops)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_non_finite_keys_reach_those_who_see_them(ops, bad, D):
    """A NaN or infinite score makes the rows that see it NaN, whatever its column and
    its request's form (few rows, one tile, a pair, divided over CTAs), and no other."""
    x = Paged([(300, 1), (290, 4), (290, 15), (200, 100), (6000, 2)], 28, 4, D, 64, BF, seed=12)
    x.q[..., 0] = x.q[..., 0].abs() + 0.1  # (the score is +inf, not -inf)
    lse0, lse = torch.empty(x.q.shape[:2], device="cuda"), torch.empty(x.q.shape[:2], device="cuda")
    good = x.call(ops, lse=lse0)
    for key in (0, 1, 2, 3, 4, 5, 62, 67, 130, 131, 132, 259, 290, 291, 295, 299, 300):
        k = x.k.clone()
        want, wlse, at = good.clone(), lse0.clone(), 0
        for b, (past, n) in enumerate(x.pairs):
            if key < past + n:
                k[x.table[b, key // 64].item(), 1, key % 64, 0] = bad
                first = max(0, key - past)  # the first of its tokens that sees it
                want[at + first:at + n, 7:14] = math.nan
                wlse[at + first:at + n, 7:14] = math.nan
            at += n
        out = ops.paged_attention(x.q, k, x.v, x.table, x.cu, x.kv_lens, lse=lse)
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(lse.isnan(), wlse.isnan()), key
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), key
        assert torch.equal(lse.nan_to_num(7.0), wlse.nan_to_num(7.0)), key
    _no_device_error(ops)


@pytest.mark.parametrize("max_tokens", [0, 16, 2000])
def test_update_after_a_length_of_2_31(ops, max_tokens):
    """Requests behind refused ones whose lengths add up beyond 32 bits are served in
    full: their pages are those that were taken."""
    big = 2 ** 31 - 1
    table, held = torch.full((4, 8), -1, dtype=torch.int32, device="cuda"), _i32([0, 0, 0, 0])
    free, n_free = torch.arange(8, dtype=torch.int32, device="cuda"), _i32([8])
    cu, kv, slots, pos, ok = ops.paged_update(_i32([0, 0, 0, 16]), _i32([big, 5, big, 33]), table, held, free, n_free,
                                              16, max_tokens)
    assert ops.device_error() == 3
    assert ok.tolist() == [0, 1, 0, 1] and kv.tolist() == [0, 5, 0, 49]
    assert held.tolist() == [0, 1, 0, 4] and n_free.tolist() == [3]
    assert sorted(table[table >= 0].tolist()) == [3, 4, 5, 6, 7]
    assert cu.tolist() == [0, big, big, big, big] and (slots == -1).all() and (pos == -1).all()
    _no_device_error(ops)


def test_update_tables_alone(ops):
    """max_tokens 0: the tables without slots, for any number of new tokens."""
    table, held = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), _i32([0, 0])
    free, n_free = torch.arange(8, dtype=torch.int32, device="cuda"), _i32([8])
    cu, kv, slots, pos, ok = ops.paged_update(_i32([0, 0]), _i32([20, 3]), table, held, free, n_free, 16, 0)
    assert cu.tolist() == [0, 20, 23] and kv.tolist() == [20, 3] and ok.tolist() == [1, 1]
    assert table[:, :2].tolist() == [[7, 6], [5, -1]] and slots.numel() == pos.numel() == 0
    _no_device_error(ops)


def test_queries_beyond_32_bits(ops):
    """More than 2^31 elements of queries, outputs and qkv rows in one call."""
    Hq, Hkv, D, page, n, B = 28, 4, 128, 64, 81300, 8  # 2.33e9 elements
    T, L = B * n, 100
    blocks = -(-L // page)
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.empty(T, (Hq + 2 * Hkv) * D, dtype=BF, device="cuda")
    k = torch.randn(B * blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    v = torch.randn(B * blocks, Hkv, page, D, generator=g, device="cuda").to(BF)
    table = torch.arange(B * blocks, dtype=torch.int32, device="cuda").view(B, blocks)
    rows = [0, 1, n - 1, n, T // 2, T - 36, T - 2, T - 1]
    qkv.view(T, -1)[rows] = torch.randn(len(rows), qkv.shape[1], generator=g, device="cuda").to(BF)
    cos, sin = _rope_tables(4, D, BF)
    q = torch.full((T, Hq, D), 7.0, dtype=BF, device="cuda")
    pos, slots = torch.full((T,), -1, dtype=torch.int32, device="cuda"), torch.full((T,), -1, dtype=torch.int32, device="cuda")
    pos[rows] = 0  # (no rotation)
    slots[T - 1] = (B - 1) * blocks * page + 99
    ops.paged_rope_append(qkv, pos, slots, cos, sin, q, k, v)
    new = qkv[rows].view(len(rows), -1, D)
    assert torch.equal(q[rows], new[:, :Hq]) and (q[[2, n + 1, T - 3]] == 7).all()
    at = ((B - 1) * blocks + 1, slice(None), 99 - 64)
    assert torch.equal(k[at], new[-1, Hq:Hq + Hkv]) and torch.equal(v[at], new[-1, Hq + Hkv:])
    del qkv
    cu, kv = _i32([n * b for b in range(B + 1)]), _i32([L] * B)
    out = torch.full_like(q, 3.0)
    ops.paged_attention(q, k, v, table, cu, kv, causal=False, out=out)
    for r in rows + [5, T - 7]:
        b = r // n
        kk = k[table[b].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :L].double().repeat_interleave(7, 0)
        vv = v[table[b].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :L].double().repeat_interleave(7, 0)
        s = torch.einsum("hd,hld->hl", q[r].double(), kk) / math.sqrt(D)
        p = torch.softmax(s, -1)
        ref, A = torch.einsum("hl,hld->hd", p, vv), torch.einsum("hl,hld->hd", p, vv.abs())
        assert ((out[r].double() - ref).abs() <= 1.02 * 2.0 ** -8 * (ref.abs() + A)).all(), r
    ops.paged_attention(q, k, v, table, cu, kv, out=out)  # causal: the last 100 tokens of each see keys
    seen = [n - L, n - 1, T - L, T - 1]
    assert (out[[0, n - L - 1, T - L - 1]] == 0).all()
    assert torch.equal(out[[n - L, T - L]][:, ::7], v[table[[0, B - 1], 0].long(), :, 0]) and (out[seen] != 0).any(-1).all()
    _no_device_error(ops)


@pytest.mark.parametrize("new,D,dtype", [(1, 64, FP), (4, 128, FP), (12, 64, FP), (36, 64, FP), (36, 128, BF)])
def test_sums_over_a_million_keys(ops, new, D, dtype):
    """2^20 keys in one CTA (few rows, one tile, a pair): the sums do not drift.  150
    requests on the same pages, the later pages' scores above the earlier ones'.

    A CTA's stream adds 16 keys at a time to a 32-bit sum, cut off (2^-23 of it each
    time at most), starts anew every 512 blocks of 128 keys and rounds once there:
    4096 2^-23 + 32 2^-24 = 4.9e-4 relative, of same-signed values; l lags by 64 per
    2^20 / 128 / 2 and thread at most, 2^-24 each and both ways: 2.5e-4.  Besides, the
    rounding of the output, e / 2, and of the probabilities: e / 2 of sum p |v| = ref,
    in full, as a key that comes again has the same error each time (a few of the 1024
    keys can hold nearly all of a row's weight, so nothing averages out)."""
    L, page, G = 1 << 20, 256, 7
    g = torch.Generator(device="cuda").manual_seed(new)
    k = torch.randn(4, 1, page, D, generator=g, device="cuda")
    k[:2] *= 0.2
    k = k.to(dtype)
    v = (torch.rand(4, 1, page, D, generator=g, device="cuda") + 0.5).to(dtype)
    v[..., 0] = 1
    blocks, B = L // page, 150
    ids = torch.arange(blocks, device="cuda")
    row = torch.where(ids < blocks * 5 // 8, ids % 2, 2 + ids % 2).int()
    q = (3 * torch.randn(B * new, G, D, generator=g, device="cuda")).to(dtype)
    lse = torch.empty(B * new, G, device="cuda")
    cu, kv = torch.arange(0, B * new + 1, new, device="cuda").int(), torch.full((B,), L - 100, device="cuda").int()
    out = ops.paged_attention(q, k, v, row.expand(B, -1).contiguous(), cu, kv, causal=False, lse=lse).double()
    count = torch.stack([(row == i).sum() for i in range(4)]).double()[:, None].expand(4, page).clone()
    count[row[-1].long(), page - 100:] -= 1
    s = torch.einsum("nhd,pkd->nhpk", q.double(), k[:, 0].double()) / math.sqrt(D)
    m = s.amax((-1, -2), keepdim=True)
    w = torch.exp(s - m) * count
    l = w.sum((-1, -2))
    ref = torch.einsum("nhpk,pkd->nhd", w, v[:, 0].double()) / l[..., None]
    e = torch.finfo(dtype).eps
    assert ((out - ref).abs() <= (7.4e-4 + e / 2 + e / 2) * ref).all(), ((out - ref).abs() / ref).max().item()
    assert ((lse.double() - (l.log() + m[..., 0, 0])).abs() <= 2.5e-4 + 30 * 2.0 ** -22).all()
    _no_device_error(ops)
