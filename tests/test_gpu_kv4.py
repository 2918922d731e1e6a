"""The paged 4-bit KV cache and the check of drafted tokens, on the GPU,
against plain implementations: whole numbers and cache bytes exactly, RoPE'd
q bit for bit, attention against its definition in 64 bits.

Attention's tolerance, relative to the largest |value| a row can see: the two
fp16 terms of q and of the probabilities leave 2^-22 of each, the score's fp32
arithmetic a few 2^-24 of a score of at most about 40 in log2 units, the
exponential 2^-22, and the sums in fp32 some 2^-22 more: below 1e-5 in all.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ATTN_TOL = 1e-5


@pytest.fixture(scope="module")
def be(tb, cuda):
    return tb.Backend(0)


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _np(t):
    return t.detach().cpu().numpy()


def _up(n, m):
    return -(-n // m)


# --- the row format, in fp32 numpy ------------------------------------------
def _bf16_rn(x):
    b = x.astype(np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) & np.uint32(0xFFFF0000)).view(np.float32)


def quantize_rows(x):
    """(codes + 8 as ints [..., D], scale, zero) of fp32 rows."""
    x = np.asarray(x, np.float32)
    mn, mx = x.min(-1), x.max(-1)
    f = np.float32
    with np.errstate(all="ignore"):
        zero = _bf16_rn(mn * f(7 / 15) + mx * f(8 / 15))
        s = np.maximum((zero - mn) * f(0.125), (mx - zero) * f(1 / 7))
        scale = ((s.view(np.uint32) + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(f)
        c = np.rint((x - zero[..., None]) / np.where(scale > 0, scale, f(1))[..., None])
        u = np.where(scale[..., None] > 0, np.clip(c, -8, 7), 0)
        finite = np.isfinite(x).all(-1)
        u = np.where(finite[..., None], u, 0).astype(np.int64) + 8
        scale, zero = np.where(finite, scale, f("nan")), np.where(finite, zero, f("nan"))
    return u, scale.astype(f), zero.astype(f)


def values_of(u, scale, zero):
    return (zero[..., None] + scale[..., None] * (u - 8).astype(np.float32)).astype(np.float32)


def rope(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1)


def _rows(rng, T, heads, D):
    x = rng.standard_normal((T, heads, D)).astype(np.float32)
    x[..., 3] *= 9  # a loud channel
    return x


# --- append and read ----------------------------------------------------------
@pytest.mark.parametrize("T,H,Hkv,D,block", [(1, 4, 4, 32, 16), (7, 8, 2, 64, 16), (33, 32, 32, 128, 32),
                                             (100, 6, 2, 128, 48), (5, 8, 1, 32, 128), (17, 3, 3, 64, 64)])
@pytest.mark.parametrize("layout", ["fused", "odd", "plain"])
def test_append_and_read_bit_exact(be, cuda, T, H, Hkv, D, block, layout):
    rng = np.random.default_rng(T * 100 + D + block)
    import torch

    q, k, v = _rows(rng, T, H, D), _rows(rng, T, Hkv, D), _rows(rng, T, Hkv, D)
    k[0, 0], v[T // 2, -1] = 0.0, 2.625  # constant rows
    NB = _up(T, block) + 2
    slots = rng.permutation(NB * block)[:T].astype(np.int32)
    pos = rng.integers(0, 500, T).astype(np.int32)
    cos, sin = be.RoPETables(D, 500, 10000.0)
    if layout == "fused":  # slices of one projection's rows
        f = _dev(np.concatenate([q, k, v], 1))
        dq, dk, dv = f[:, :H], f[:, H:H + Hkv], f[:, H + Hkv:]
    elif layout == "odd":  # rows that no 16-byte load reaches
        f = torch.empty(T * ((H + 2 * Hkv) * D + 1) + 1, device=cuda)[1:]
        f = f.view(T, (H + 2 * Hkv) * D + 1)[:, : (H + 2 * Hkv) * D].unflatten(1, (H + 2 * Hkv, D))
        f.copy_(_dev(np.concatenate([q, k, v], 1)))
        dq, dk, dv = f[:, :H], f[:, H:H + Hkv], f[:, H + Hkv:]
    else:
        dq, dk, dv = _dev(q), _dev(k), _dev(v)
    pages = be.KV4Pages(NB, Hkv, D, block)
    qr = be.KV4AppendRoPE(pages, dk, dv, _dev(cos), _dev(sin), _dev(pos), _dev(slots), q=dq)
    c, s = cos[pos][:, None], sin[pos][:, None]
    np.testing.assert_array_equal(_np(qr), rope(q, c, s))
    gk, gv = (_np(t) for t in be.KV4Read(pages, _dev(slots)))
    for got, x in ((gk, rope(k, c, s)), (gv, v)):
        u, scale, zero = quantize_rows(x)
        np.testing.assert_array_equal(got, values_of(u, scale, zero))
        # every value within half a scale of what is held, but for the rounding of the sums
        assert (np.abs(got.astype(np.float64) - x) <= 0.5 * scale[..., None] * (1 + 1e-5) + 1e-6 * np.abs(x)).all()
    # the bytes are the documented layout
    raw = _np(pages)
    u, scale, zero = quantize_rows(v)
    for t in range(0, T, max(1, T // 5)):
        blk, off = divmod(int(slots[t]), block)
        tile, r = raw[blk, :, off // 16], off % 16
        np.testing.assert_array_equal(tile[:, 8 * D + r * (D // 2): 8 * D + (r + 1) * (D // 2)],
                                      (u[t, :, 0::2] | u[t, :, 1::2] << 4).astype(np.uint8))
        w = tile[:, 16 * D + 64 + 4 * r: 16 * D + 68 + 4 * r].copy().view(np.uint32)[:, 0]
        np.testing.assert_array_equal(w, zero[t].view(np.uint32) | scale[t].view(np.uint32) >> 16)


def test_append_extremes(be, cuda):
    """Rows at the ends of fp32, with an offset far larger than their range, and rows that are not finite."""
    rng = np.random.default_rng(5)
    T, D = 9, 64
    v = rng.standard_normal((T, 1, D)).astype(np.float32)
    v[0] *= np.float32(1e37)
    v[1] *= np.float32(1e-36)
    v[2] = 100 + np.float32(0.01) * v[2]
    v[3] = np.float32(1e-42) * np.sign(v[3])  # subnormal
    v[4, 0, 5] = np.nan
    v[5, 0, 63] = np.inf
    v[6, 0, 0] = -np.inf
    v[7] = np.where(np.arange(D) % 2, np.float32(3e38), np.float32(-3e38))
    pages = be.KV4Pages(1, 1, D, 16)
    slots = _dev(np.arange(T, dtype=np.int32))
    assert be.KV4AppendRoPE(pages, _dev(v), _dev(v), None, None, None, slots) is None
    gk, gv = (_np(t) for t in be.KV4Read(pages, slots))
    u, scale, zero = quantize_rows(v)
    np.testing.assert_array_equal(gk, values_of(u, scale, zero))
    np.testing.assert_array_equal(gv, gk)
    assert np.isnan(gv[4:7]).all() and np.isfinite(gv[[0, 1, 2, 3, 7, 8]]).all()


def test_append_padding_and_bad_slots(be, cuda):
    import torch

    rng = np.random.default_rng(6)
    T, H, Hkv, D = 6, 4, 2, 32
    q, k, v = _rows(rng, T, H, D), _rows(rng, T, Hkv, D), _rows(rng, T, Hkv, D)
    cos, sin = be.RoPETables(D, 50, 10000.0)
    pages = be.KV4Pages(2, Hkv, D, 16)
    pages.fill_(0xA5)
    before = pages.clone()
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots = np.array([-1, 32, 3, 4, 5, -1], np.int32)  # padding, past the cache, stored, bad positions, padding
    pos = np.array([0, 1, 2, 50, -1, 3], np.int32)
    qr = _np(be.KV4AppendRoPE(pages, _dev(k), _dev(v), _dev(cos), _dev(sin), _dev(pos), _dev(slots), q=_dev(q),
                              bad=bad))
    assert int(bad) == 3
    for t in (0, 2, 5):
        np.testing.assert_array_equal(qr[t], rope(q[t], cos[pos[t]], sin[pos[t]]))
    assert (qr[[1, 3, 4]] == 0).all()
    diff = (pages != before).view(2, Hkv, -1).any(-1).cpu().numpy()
    assert diff[0].all() and not diff[1].any()
    k2, v2 = (_np(t) for t in be.KV4Read(pages, _dev(np.array([-1, 3, 99], np.int32))))
    assert (k2[[0, 2]] == 0).all() and (v2[[0, 2]] == 0).all()
    np.testing.assert_array_equal(v2[1], values_of(*quantize_rows(v[2])))


# --- plan -----------------------------------------------------------------------
def plan_ref(held, ctx, new, table, free, count, T, bs):
    """The plan request by request with a Python stack."""
    B, cols = table.shape
    have, need = [_up(h, bs) for h in held], [_up(c + n, bs) for c, n in zip(ctx, new)]
    give = [table[b, need[b]:have[b]].tolist() for b in range(B) if min(held[b], ctx[b], new[b]) >= 0]
    take = sum(max(0, n - h) for h, n in zip(have, need))
    room = count + sum(map(len, give))
    bad = (any(min(x) < 0 for x in zip(held, ctx, new)) or max(have + need, default=0) > cols or room > len(free)
           or take > room or sum(new) > T)
    pos, slots = np.zeros(T, np.int32), np.full(T, -1, np.int32)
    if bad:
        return np.zeros(B + 1, np.int32), np.array(ctx), pos, slots, count, table, free, 1
    table, stack = table.copy(), free[:count].tolist()
    for g in give:
        stack += g
    free = free.copy()
    free[: len(stack)] = stack
    for b in range(B):
        for j in range(have[b], need[b]):
            table[b, j] = stack.pop()
    starts, t = [0], 0
    for b in range(B):
        for i in range(new[b]):
            p = ctx[b] + i
            pos[t], slots[t] = p, table[b, p // bs] * bs + p % bs
            t += 1
        starts.append(t)
    return np.array(starts), np.array(ctx) + np.array(new), pos, slots, len(stack), table, free, 0


def _plan_state(rng, held, bs, cols, spare):
    have = [_up(h, bs) for h in held]
    total = sum(have) + spare
    order = rng.permutation(total).astype(np.int32)
    table = np.full((len(held), cols), -1, np.int32)
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = order[at:at + n]
        at += n
    free = np.full(total, -7, np.int32)
    free[: total - at] = order[at:]
    return table, free, total - at


def _check_plan(be, held, ctx, new, table, free, count, T, bs):
    want = plan_ref(held, ctx, new, table, free, count, T, bs)
    i32 = lambda a: _dev(np.asarray(a, np.int32))  # noqa: E731
    dt, df = i32(table), i32(free)
    p = be.KV4Plan(i32(held), i32(ctx), i32(new), dt, df, i32([count]), T, bs)
    again = be.KV4Plan(i32(held), i32(ctx), i32(new), dt, df, i32([count]), T, bs)  # nothing of a launch's own is read
    for s in (p, again):
        got = (s.q_start, s.seq_lens, s.positions, s.slots, s.free_count, dt, df, s.bad)
        names = ("q_start", "seq_lens", "positions", "slots", "free_count", "block_table", "free_list", "bad")
        for name, g, w in zip(names, got, want):
            np.testing.assert_array_equal(_np(g).ravel(), np.asarray(w).ravel(), err_msg=name)
    return want


@pytest.mark.parametrize("B,bs,most", [(1, 16, 40), (3, 16, 100), (64, 32, 300), (513, 16, 60), (1500, 64, 900),
                                       (5000, 16, 30)])
def test_plan_matches_a_stack(be, cuda, B, bs, most):
    rng = np.random.default_rng(B + bs)
    held = rng.integers(0, most, B)
    ctx = np.where(rng.random(B) < 0.3, (held * rng.random(B)).astype(int), held)  # rolled back
    ctx[rng.random(B) < 0.1] = 0  # finished
    new = np.where(rng.random(B) < 0.5, 1, rng.integers(0, most, B))
    new[rng.random(B) < 0.1] = 0
    held, ctx, new = held.tolist(), ctx.tolist(), new.tolist()
    cols = _up(2 * most, bs) + 2
    table, free, count = _plan_state(rng, held, bs, cols, sum(_up(c + n, bs) for c, n in zip(ctx, new)) + 5)
    want = _check_plan(be, held, ctx, new, table, free, count, sum(new) + 9, bs)
    assert want[-1] == 0


def test_plan_refuses_as_a_whole(be, cuda):
    rng = np.random.default_rng(9)
    held, ctx, new = [20, 33, 0], [20, 10, 0], [1, 1, 40]
    table, free, count = _plan_state(rng, held, 16, 4, 1)
    good = _check_plan(be, held, ctx, new, table, free, count, 42, 16)  # 3 pages wanted, 2 given back, 1 free
    assert good[-1] == 0 and good[4] == 0
    short = _check_plan(be, held, ctx, [1, 1, 49], table, free, count, 60, 16)  # one page more than there is
    assert short[-1] == 1
    assert _check_plan(be, held, ctx, new, table, free, count, 41, 16)[-1] == 1  # token rows
    assert _check_plan(be, held, ctx, [50, 1, 0], table, free, count, 60, 16)[-1] == 1  # table columns
    assert _check_plan(be, held, [20, 10, -1], new, table, free, count, 60, 16)[-1] == 1
    assert _check_plan(be, [20, 33, 0], [20, 33, 0], [0, 0, 0], table, free, count, 0, 16)[-1] == 0


def test_plan_refuses_more_pages_than_there_are(be, cuda):
    """Lengths that only a broken caller gives: pages past the pool's, sums past 32 bits."""
    rng = np.random.default_rng(10)
    big = 2**31 - 1
    for held, ctx, new in (([big - 5], [big - 5], [3]), ([big], [big], [1]), ([big], [0], [1]), ([0], [big], [big]),
                           ([200], [200], [1])):
        table, free = np.zeros((1, 300), np.int32), np.arange(9, dtype=np.int32)
        step = be.KV4Plan(_dev(np.array(held, np.int32)), _dev(np.array(ctx, np.int32)),
                          _dev(np.array(new, np.int32)), _dev(table), _dev(free), _dev(np.array([9], np.int32)), 4, 16)
        assert int(step.bad) == 1 and int(step.free_count) == 9 and (_np(step.slots) == -1).all()


def test_plan_of_nothing(be, cuda):
    table, free = np.zeros((0, 4), np.int32), np.arange(6, dtype=np.int32)
    want = _check_plan(be, [], [], [], table, free, 6, 5, 16)
    assert want[-1] == 0


# --- attention --------------------------------------------------------------------
class Cache:
    """Requests' K and V in a 4-bit cache whose every other byte is garbage (NaN words included)."""

    def __init__(self, be, rng, lens, Hkv, D, block, cols_more=2, spread=1.0):
        import torch

        self.lens, self.block = list(lens), block
        have = [_up(n, block) for n in lens]
        NB = sum(have) + 3
        order = rng.permutation(NB).astype(np.int32)
        self.table = np.full((len(lens), max(have + [0]) + cols_more), -1, np.int32)
        self.table[:, :] = rng.integers(-5, NB + 5, self.table.shape)  # past a request's pages: anything
        self.pages = be.KV4Pages(NB, Hkv, D, block)
        self.pages.copy_(torch.from_numpy(rng.integers(0, 256, tuple(self.pages.shape), np.uint8)))
        self.pages[..., 16 * D:] = 0xFF  # NaN scales and zeros
        at = 0
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            self.table[b, : have[b]] = order[at:at + have[b]]
            at += have[b]
            k, v = spread * _rows(rng, n, Hkv, D), _rows(rng, n, Hkv, D)
            j = np.arange(n)
            slots = (self.table[b, j // block] * block + j % block).astype(np.int32)
            if n:
                be.KV4AppendRoPE(self.pages, _dev(k), _dev(v), None, None, None, _dev(slots))
            self.k.append(values_of(*quantize_rows(k)).astype(np.float64))
            self.v.append(values_of(*quantize_rows(v)).astype(np.float64))


def attend_ref(cache, q, new, scale):
    out, most, row = np.zeros(q.shape), np.zeros(q.shape[0]), 0
    G = q.shape[1] // cache.k[0].shape[1]
    for b, n in enumerate(new):
        length = cache.lens[b]
        for i in range(n):
            seen = length - n + i + 1
            if seen > 0:
                k, v = np.repeat(cache.k[b][:seen], G, 1), np.repeat(cache.v[b][:seen], G, 1)
                s = np.einsum("hd,jhd->hj", q[row].astype(np.float64), k) * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[row] = np.einsum("hj,jhd->hd", p, v)
                most[row] = np.abs(v).max()
            row += 1
    return out, most


def _check_attention(be, cache, q, new, scale=None, max_q=None, view=None, bad=None):
    D = q.shape[-1]
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    got = be.KV4Attention(_dev(q) if view is None else view, cache.pages, _dev(cache.table),
                          _dev(np.array(cache.lens, np.int32)), _dev(starts), max_q or max(new + [1]), scale, bad=bad)
    want, most = attend_ref(cache, q, new, scale or 1 / math.sqrt(D))
    got = _np(got).astype(np.float64)
    assert np.isfinite(got).all()
    err = np.abs(got - want).max((1, 2)) if len(got) else np.zeros(0)
    assert (err <= ATTN_TOL * most).all(), (err / np.maximum(most, 1e-30)).max()
    return got


@pytest.mark.parametrize("H,Hkv,D,block", [(4, 4, 128, 16), (8, 2, 128, 32), (16, 2, 128, 16), (3, 1, 64, 16),
                                           (8, 1, 64, 48), (12, 2, 32, 64), (2, 2, 32, 16), (20, 2, 128, 128)])
@pytest.mark.parametrize("new", [1, 2, 5, 40])
def test_attention_ragged(be, cuda, H, Hkv, D, block, new):
    rng = np.random.default_rng(H * 1000 + D + new)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 129, 500, 1111]
    news = [min(new, n) for n in lens]
    cache = Cache(be, rng, lens, Hkv, D, block)
    q = rng.standard_normal((sum(news), H, D)).astype(np.float32)
    _check_attention(be, cache, q, news)


def test_attention_of_more_rows_than_announced(be, cuda):
    rng = np.random.default_rng(28)
    lens, news = [300, 90, 5], [40, 90, 1]
    cache = Cache(be, rng, lens, 2, 64, 16)
    q = rng.standard_normal((sum(news), 8, 64)).astype(np.float32)
    for max_q in (1, 3, 20):
        _check_attention(be, cache, q, news, max_q=max_q)


def test_attention_long_and_one_of_each(be, cuda):
    rng = np.random.default_rng(11)
    lens = [20011, 3, 9000]
    cache = Cache(be, rng, lens, 2, 128, 16)
    q = rng.standard_normal((3, 16, 128)).astype(np.float32) * 3
    _check_attention(be, cache, q, [1, 1, 1])
    q = rng.standard_normal((70, 16, 128)).astype(np.float32)
    _check_attention(be, cache, q, [2, 3, 65])


def test_attention_empty_rows_and_requests(be, cuda):
    """No new tokens, an empty cache, more rows than cached positions, rows of no request."""
    import torch

    rng = np.random.default_rng(12)
    lens, news = [0, 50, 3, 0, 70, 9], [2, 0, 5, 0, 1, 9]
    cache = Cache(be, rng, lens, 2, 64, 16)
    q = rng.standard_normal((sum(news), 4, 64)).astype(np.float32)
    got = _check_attention(be, cache, q, news)
    assert (got[:4] == 0).all() and np.abs(got[4]).max() > 0  # two rows without keys, two before the first of three
    starts = _dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32))
    more = torch.cat([_dev(q), torch.full((5, 4, 64), float("nan"), device=cuda)])
    out = be.KV4Attention(more, cache.pages, _dev(cache.table), _dev(np.array(lens, np.int32)), starts, 9)
    np.testing.assert_array_equal(_np(out[: len(q)]), got.astype(np.float32))
    assert (out[len(q):] == 0).all()
    none = be.KV4Attention(more[:0], cache.pages, _dev(cache.table), _dev(np.array(lens, np.int32)),
                           torch.zeros(7, dtype=torch.int32, device=cuda), 1)
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("amp", [1e-30, 1e-3, 30.0, 300.0])
def test_attention_scales(be, cuda, amp):
    """Values of very different sizes in one request, and scores from all equal to one-hot."""
    import torch

    rng = np.random.default_rng(13)
    n, D = 300, 128
    cache = Cache(be, rng, [n], 1, D, 16)
    v = _rows(rng, n, 1, D) * np.exp(rng.uniform(-12, 12, (n, 1, 1))).astype(np.float32)
    slots = (cache.table[0, np.arange(n) // 16] * 16 + np.arange(n) % 16).astype(np.int32)
    k = values_of(*quantize_rows(cache.k[0].astype(np.float32)))
    be.KV4AppendRoPE(cache.pages, _dev(k), _dev(v), None, None, None, _dev(slots))
    gk, gv = be.KV4Read(cache.pages, _dev(slots))
    cache.k[0], cache.v[0] = _np(gk).astype(np.float64), _np(gv).astype(np.float64)
    q = (amp * rng.standard_normal((2, 4, D))).astype(np.float32)
    starts = torch.tensor([0, 2], dtype=torch.int32, device=cuda)
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)), starts, 2))
    want, most = attend_ref(cache, q, [2], 1 / math.sqrt(D))
    # a score of s is off by about 2^-22 |s| in log2 units: amp 300 makes scores of some 10^4
    tol = ATTN_TOL * max(1.0, amp)
    assert (np.abs(got - want).max((1, 2)) <= tol * most).all()


def test_attention_nan_rows_stay_where_they_are(be, cuda):
    """A cached row that is not finite makes NaN of the rows that see it and of no other."""
    rng = np.random.default_rng(14)
    n, D = 40, 64
    for part in (0, 1):
        cache = Cache(be, rng, [n, n], 2, D, 16)
        x = [_rows(rng, 1, 2, D), _rows(rng, 1, 2, D)]
        x[part][0, 1, 7] = np.inf
        slot = np.array([cache.table[0, 38 // 16] * 16 + 38 % 16], np.int32)
        be.KV4AppendRoPE(cache.pages, _dev(x[0]), _dev(x[1]), None, None, None, _dev(slot))
        q = rng.standard_normal((8, 4, D)).astype(np.float32)
        starts = _dev(np.array([0, 4, 8], np.int32))
        got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n, n], np.int32)), starts,
                                  4))
        assert np.isnan(got[2:4, 2:]).all()  # the second kv head's rows at positions 38 and 39
        got[2:4, 2:] = 0
        assert np.isfinite(got).all()


def test_attention_bad_table_entries_are_hidden(be, cuda):
    import torch

    rng = np.random.default_rng(15)
    cache = Cache(be, rng, [100, 20], 1, 128, 32)
    cache.table[0, 1] = cache.pages.shape[0]  # positions 32 .. 63
    cache.table[1, 0] = -1
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = rng.standard_normal((2, 4, 128)).astype(np.float32)
    starts = _dev(np.array([0, 1, 2], np.int32))
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([100, 20], np.int32)), starts, 1,
                              bad=bad))
    assert int(bad) > 0
    keep = np.r_[0:32, 64:100]
    s = np.einsum("hd,jd->hj", q[0].astype(np.float64), cache.k[0][keep, 0]) / math.sqrt(128)
    p = np.exp(s - s.max(-1, keepdims=True))
    want = (p / p.sum(-1, keepdims=True)) @ cache.v[0][keep, 0]
    assert np.abs(got[0] - want).max() <= ATTN_TOL * np.abs(cache.v[0]).max()
    assert (got[1] == 0).all()


def test_attention_q_views_streams_and_repeats(be, cuda):
    """Strided and unaligned q, a stream of the caller's, and the same bits from call to call."""
    import torch

    rng = np.random.default_rng(16)
    lens, news = [333, 40], [1, 1]
    cache = Cache(be, rng, lens, 2, 128, 16)
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    fused = torch.zeros(2, 12 * 128, device=cuda)
    fused[:, : 8 * 128] = _dev(q).view(2, -1)
    got = _check_attention(be, cache, q, news, view=fused.view(2, 12, 128)[:, :8])
    odd = torch.zeros(2 * 1025 + 1, device=cuda)[1:].view(2, 1025)[:, :1024].unflatten(1, (8, 128))
    odd.copy_(_dev(q))
    np.testing.assert_array_equal(_check_attention(be, cache, q, news, view=odd), got)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = _check_attention(be, cache, q, news)
    np.testing.assert_array_equal(again, got)
    np.testing.assert_array_equal(_check_attention(be, cache, q, news, max_q=2), _check_attention(be, cache, q, news, max_q=2))


# Prompt chunks: the rows of a kv head are more than the kernel for single tokens
# and drafts takes, so another one runs (their tiles, masks and splits differ).
CHUNK = [(4, 2, 64, 16, 60), (8, 1, 128, 16, 40), (6, 2, 128, 48, 100), (8, 8, 64, 32, 300), (128, 1, 64, 16, 3),
         (4, 1, 32, 16, 60), (8, 8, 32, 48, 200)]


@pytest.mark.parametrize("H,Hkv,D,block,new", CHUNK)
def test_attention_chunks(be, cuda, H, Hkv, D, block, new):
    """Chunks at the ends of tiles and units, beside requests of one token and of none."""
    rng = np.random.default_rng(100 * H + new)
    lens = [new, new + 1, 63, 64, 65, 128, 257, 700, 0, 1, 2000]
    news = [min(n, m) for n, m in zip(lens, [new, new, new, new, new - 1, 1, new, new, new, new, new])]
    news[8] = 0
    cache = Cache(be, rng, lens, Hkv, D, block)
    q = rng.standard_normal((sum(news), H, D)).astype(np.float32)
    _check_attention(be, cache, q, news)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_chunk_empty_rows(be, cuda, D):
    """More new rows than cached positions (the first see nothing), an empty cache, rows of no request."""
    import torch

    rng = np.random.default_rng(21)
    lens, news = [0, 150, 3, 0, 70, 200, 130], [80, 0, 70, 0, 71, 200, 1]
    cache = Cache(be, rng, lens, 1, D, 16)
    q = rng.standard_normal((sum(news), 2, D)).astype(np.float32)
    got = _check_attention(be, cache, q, news)
    assert (got[:80 + 67] == 0).all() and np.abs(got[80 + 67]).max() > 0
    starts = _dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32))
    more = torch.cat([_dev(q), torch.full((5, 2, D), float("nan"), device=cuda)])
    out = be.KV4Attention(more, cache.pages, _dev(cache.table), _dev(np.array(lens, np.int32)), starts, 200)
    np.testing.assert_array_equal(_np(out[: len(q)]), got.astype(np.float32))
    assert (out[len(q):] == 0).all()


@pytest.mark.parametrize("amp", [1e-30, 1e-3, 30.0, 300.0])
def test_attention_chunk_scales(be, cuda, amp):
    rng = np.random.default_rng(22)
    n, D = 300, 128
    cache = Cache(be, rng, [n], 1, D, 16)
    v = _rows(rng, n, 1, D) * np.exp(rng.uniform(-12, 12, (n, 1, 1))).astype(np.float32)
    slots = (cache.table[0, np.arange(n) // 16] * 16 + np.arange(n) % 16).astype(np.int32)
    be.KV4AppendRoPE(cache.pages, _dev(cache.k[0].astype(np.float32)), _dev(v), None, None, None, _dev(slots))
    gk, gv = be.KV4Read(cache.pages, _dev(slots))
    cache.k[0], cache.v[0] = _np(gk).astype(np.float64), _np(gv).astype(np.float64)
    q = (amp * rng.standard_normal((150, 4, D))).astype(np.float32)
    starts = _dev(np.array([0, 150], np.int32))
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)), starts, 150))
    want, most = attend_ref(cache, q, [150], 1 / math.sqrt(D))
    # a score of s is off by about 2^-22 |s| in log2 units: amp 300 makes scores of some 10^4
    assert (np.abs(got - want).max((1, 2)) <= ATTN_TOL * max(1.0, amp) * most).all()


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("new", [70, 128, 129])
def test_attention_chunk_lengths_and_sizes_of_values(be, cuda, D, new):
    """Many tiles to a CTA around 128 rows, values whose size grows along the context and jumps."""
    rng = np.random.default_rng(27)
    lens, news = [3000, 2500, 140, 1900], [new, new - 1, new, 1]
    cache = Cache(be, rng, lens, 8, D, 64)
    for b, n in enumerate(lens):
        size = np.exp(8 * np.arange(n) / n + 3 * rng.standard_normal(n)).astype(np.float32)
        v = _rows(rng, n, 8, D) * size[:, None, None]
        j = np.arange(n)
        slots = (cache.table[b, j // 64] * 64 + j % 64).astype(np.int32)
        be.KV4AppendRoPE(cache.pages, _dev(cache.k[b].astype(np.float32)), _dev(v), None, None, None, _dev(slots))
        gk, gv = be.KV4Read(cache.pages, _dev(slots))
        cache.k[b], cache.v[b] = _np(gk).astype(np.float64), _np(gv).astype(np.float64)
    q = rng.standard_normal((sum(news), 8, D)).astype(np.float32)
    _check_attention(be, cache, q, news)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("part", [0, 1])
def test_attention_chunk_nan_rows_stay_where_they_are(be, cuda, D, part):
    rng = np.random.default_rng(23)
    n, new = 200, 70
    cache = Cache(be, rng, [n, n], 2, D, 16)
    x = [_rows(rng, 1, 2, D), _rows(rng, 1, 2, D)]
    x[part][0, 1, 7] = np.inf
    slot = np.array([cache.table[0, 180 // 16] * 16 + 180 % 16], np.int32)
    be.KV4AppendRoPE(cache.pages, _dev(x[0]), _dev(x[1]), None, None, None, _dev(slot))
    q = rng.standard_normal((2 * new, 4, D)).astype(np.float32)
    starts = _dev(np.array([0, new, 2 * new], np.int32))
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n, n], np.int32)), starts, new))
    assert np.isnan(got[50:70, 2:]).all()  # the second kv head's rows from position 180 on
    got[50:70, 2:] = 0
    assert np.isfinite(got).all()


def test_attention_chunk_bad_table_entries_are_hidden(be, cuda):
    import torch

    rng = np.random.default_rng(24)
    n, new, D = 200, 80, 128
    cache = Cache(be, rng, [n], 1, D, 32)
    cache.table[0, 1] = cache.pages.shape[0]  # positions 32 .. 63
    cache.table[0, 5] = -1                    # and 160 .. 191
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = rng.standard_normal((new, 4, D)).astype(np.float32)
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)),
                              _dev(np.array([0, new], np.int32)), new, bad=bad))
    assert int(bad) > 0
    for i in range(new):
        seen = np.arange(n - new + i + 1)
        seen = seen[(seen // 32 != 1) & (seen // 32 != 5)]
        s = np.einsum("hd,jd->hj", q[i].astype(np.float64), cache.k[0][seen, 0]) / math.sqrt(D)
        p = np.exp(s - s.max(-1, keepdims=True))
        want = (p / p.sum(-1, keepdims=True)) @ cache.v[0][seen, 0]
        assert np.abs(got[i] - want).max() <= ATTN_TOL * np.abs(cache.v[0]).max()


def test_attention_chunk_q_views_streams_and_repeats(be, cuda):
    import torch

    rng = np.random.default_rng(25)
    lens, news = [333, 90], [100, 20]
    cache = Cache(be, rng, lens, 2, 128, 16)
    q = rng.standard_normal((120, 8, 128)).astype(np.float32)
    fused = torch.zeros(120, 12 * 128, device=cuda)
    fused[:, : 8 * 128] = _dev(q).view(120, -1)
    got = _check_attention(be, cache, q, news, view=fused.view(120, 12, 128)[:, :8])
    odd = torch.zeros(120 * 1025 + 1, device=cuda)[1:].view(120, 1025)[:, :1024].unflatten(1, (8, 128))
    odd.copy_(_dev(q))
    np.testing.assert_array_equal(_check_attention(be, cache, q, news, view=odd), got)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = _check_attention(be, cache, q, news)
    np.testing.assert_array_equal(again, got)


@pytest.mark.parametrize("H,new", [(2, 2), (4, 2), (8, 3), (8, 80), (2, 40)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_rows_of_q_do_not_meet(be, cuda, H, new, D):
    """A row of q that is not finite, or far larger or smaller than the others, changes its own output only."""
    rng = np.random.default_rng(26)
    n = 190
    cache = Cache(be, rng, [n], 1, D, 16)
    q = rng.standard_normal((new, H, D)).astype(np.float32)
    q[0, 0, 5] = np.inf
    q[0, 1] *= 1e-25
    q[1, 0] *= 1e20
    q[1, 1, D - 1] = np.nan
    if new > 2:
        q[2] *= 1e-6
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)),
                              _dev(np.array([0, new], np.int32)), new)).astype(np.float64)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1]).all()
    assert np.isfinite(got[1, 0]).all()
    rest = np.ones((new, H), bool)
    rest[0, 0] = rest[1, 0] = rest[1, 1] = False
    want, most = attend_ref(cache, np.where(rest[..., None], q, 0), [new], 1 / math.sqrt(D))
    assert np.abs(got - want)[rest].max() <= ATTN_TOL * most.max()


# --- verification of drafts -----------------------------------------------------
def verify_ref(p, x, u, q, lens):
    B, K = x.shape
    V = p.shape[2]
    f = np.float32
    tokens, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int32)
    for b in range(B):
        n = K if lens is None else min(max(int(lens[b]), 0), K)
        r = 0
        while r < n:
            t = x[b, r]
            if not (0 <= t < V) or not f(u[b, r]) * f(q[b, r, t] if q is not None else 1) < p[b, r, t]:
                break
            tokens[b, r] = t
            r += 1
        accepted[b] = r
        rest = p[b, r].copy()
        if r < n and q is not None:
            rest = rest - q[b, r]
        elif r < n and 0 <= x[b, r] < V:
            rest[x[b, r]] = 0
        for w in (rest, p[b, r]):
            with np.errstate(invalid="ignore"):
                w = np.nan_to_num(np.clip(w, 0, 1), nan=0.0).astype(np.float64)
            fixed = [int(v) for v in np.floor(w * 2.0**36)]
            if sum(fixed):
                break
        target = (sum(fixed) * int(np.floor(np.float64(u[b, K]) * 2**24))) >> 24
        ends = np.cumsum(np.array(fixed, dtype=object))
        tokens[b, r] = next((i for i, e in enumerate(ends) if e > target), 0)
    return tokens, accepted


def _probs(rng, *shape, amp=2.0):
    z = amp * rng.standard_normal(shape)
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (5, 1, 7), (3, 8, 1001), (17, 3, 4096), (2, 5, 1), (4, 0, 500),
                                   (2, 40, 63), (1, 2, 100003)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_matches_the_definition(be, cuda, B, K, V, certain):
    rng = np.random.default_rng(B * 100 + K + V)
    p = _probs(rng, B, K + 1, V)
    q = None if certain else _probs(rng, B, K, V, amp=1.0) * np.float32(0.5) + p[:, :K] * np.float32(0.5)
    x = rng.integers(0, V, (B, K))
    for b in range(B):  # likely drafts, so that several are accepted
        for i in range(K):
            if rng.random() < 0.8:
                x[b, i] = p[b, i].argmax()
    u = (rng.integers(0, 1 << 24, (B, K + 1)) / 2.0**24).astype(np.float32)
    if certain:
        u[:, :K] *= np.float32(0.05)
    for lens in (None, rng.integers(0, K + 1, B).astype(np.int32)):
        want = verify_ref(p, x, u, q, lens)
        got = be.VerifyDraft(_dev(p), _dev(x), _dev(u), None if q is None else _dev(q), None if lens is None else _dev(lens))
        np.testing.assert_array_equal(_np(got[1]), want[1])
        np.testing.assert_array_equal(_np(got[0]), want[0])


def test_verify_edges(be, cuda):
    """Equal distributions, u = 0 and the largest u, NaN and empty rows, drafts outside the vocabulary, strides."""
    import torch

    rng = np.random.default_rng(21)
    B, K, V = 6, 3, 300
    p = _probs(rng, B, K + 1, V)
    q = p[:, :K].copy()
    x = np.tile(np.array([4, 9, 11]), (B, 1))
    u = np.full((B, K + 1), 0.5, np.float32)
    u[0] = 0.0
    u[1] = 1 - 2.0**-24
    q[2] = p[2, :K] * 4  # refused, and nothing is left of p - q: the draw is from p
    u[2, :K] = 0.9
    p[3, 0, 5] = np.nan
    p[3, 0, 4] = 0.0  # refused at once; the draw skips the NaN
    x[4, 1] = V  # outside
    p[5, K] = 0.0  # all accepted, and an empty row
    p[5, :K, :] = 1.0 / V
    q[5] = 1.0 / V
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    want = verify_ref(p, x, u, q, None)
    got = be.VerifyDraft(_dev(p), _dev(x), _dev(u), _dev(q), bad=bad)
    np.testing.assert_array_equal(_np(got[1]), want[1])
    np.testing.assert_array_equal(_np(got[0]), want[0])
    assert int(bad) == 2 and want[1][4] == 1 and want[1][5] == K and want[0][5, K] == 0
    # rows of wider buffers, at every alignment
    for pad in (1, 4):
        wide = torch.zeros(B, K + 1, V + pad, device=cuda)
        wide[..., :V] = _dev(p)
        wq = torch.zeros(B, K + 1, V + pad, device=cuda)
        wq[:, :K, :V] = _dev(q)
        got = be.VerifyDraft(wide[..., :V], _dev(x), _dev(u), wq[:, :K, :V])
        np.testing.assert_array_equal(_np(got[0]), want[0])


def test_verify_draws_the_target_distribution(be, cuda):
    """Speculative sampling's promise: whatever the drafter, an emitted token follows the target.  40000 draws
    of a first token over 8 words: each count within 5 standard deviations."""
    rng = np.random.default_rng(22)
    n, V = 40000, 8
    p, q = _probs(rng, 1, 2, V)[0], _probs(rng, 1, 1, V)[0]
    q64 = q[0].astype(np.float64)
    x = rng.choice(V, (n, 1), p=q64 / q64.sum())
    u = rng.random((n, 2)).astype(np.float32)
    u[u == 1] = 0
    tokens, _ = be.VerifyDraft(_dev(np.tile(p, (n, 1, 1))), _dev(x), _dev(u), _dev(np.tile(q, (n, 1, 1))))
    counts = np.bincount(_np(tokens)[:, 0], minlength=V)
    assert (np.abs(counts - n * p[0]) <= 5 * np.sqrt(n * p[0] * (1 - p[0]))).all(), (counts, n * p[0])


# --- refusals ----------------------------------------------------------------------
def test_refusals(tb, be, cuda):
    import torch

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=cuda)  # noqa: E731
    pages = be.KV4Pages(4, 2, 64, 16)
    for args in ((4, 2, 48, 16), (4, 2, 64, 24), (4, 2, 64, 0)):
        with pytest.raises(tb.ShapeError):
            be.KV4Pages(*args)
    with pytest.raises(tb.ShapeError):  # host tensors
        be.KV4Attention(f32(1, 4, 64).cpu(), pages, i32(1, 2), i32(1), i32(2), 1)
    with pytest.raises(tb.ShapeError):  # heads on kv heads
        be.KV4Attention(f32(1, 3, 64), pages, i32(1, 2), i32(1), i32(2), 1)
    with pytest.raises(tb.ShapeError):  # head size
        be.KV4Attention(f32(1, 4, 32), pages, i32(1, 2), i32(1), i32(2), 1)
    with pytest.raises(tb.ShapeError):  # lengths of another type
        be.KV4Attention(f32(1, 4, 64), pages, i32(1, 2), i32(1).long(), i32(2), 1)
    with pytest.raises(tb.ShapeError):
        be.KV4Attention(f32(1, 4, 64), pages, i32(1, 2), i32(1), i32(1), 1)
    with pytest.raises(tb.ShapeError):  # channels that are not contiguous
        be.KV4Attention(f32(1, 64, 4).transpose(1, 2), pages, i32(1, 2), i32(1), i32(2), 1)
    with pytest.raises(tb.ShapeError):
        be.KV4AppendRoPE(pages, f32(3, 2, 64), f32(2, 2, 64), None, None, None, i32(3))
    with pytest.raises(tb.ShapeError):  # RoPE without positions
        be.KV4AppendRoPE(pages, f32(3, 2, 64), f32(3, 2, 64), f32(9, 32), f32(9, 32), None, i32(3))
    with pytest.raises(tb.ShapeError):
        be.KV4Plan(i32(2), i32(2), i32(3), i32(2, 4), i32(9), i32(1), 5, 16)
    with pytest.raises(tb.TendoB200Error) as e:  # block size
        be.KV4Plan(i32(2), i32(2), i32(2), i32(2, 4), i32(9), i32(1), 5, 24)
    assert e.value.code == tb.TB_ERROR_INVALID_ARGUMENT
    with pytest.raises(tb.ShapeError):
        be.VerifyDraft(f32(2, 3, 9), i32(2, 3).long(), f32(2, 4))
    with pytest.raises(tb.ShapeError):
        be.VerifyDraft(f32(2, 4, 9), i32(2, 3), f32(2, 4))
    # at the C entry points
    s = torch.cuda.current_stream().cuda_stream
    out, q, ws = f32(1, 4, 64), f32(1, 4, 64), f32(1 << 22)
    table, lens, starts = i32(1, 2), i32(1), i32(2)

    def attention(D=64, H=4, block=16, ws_ptr=ws.data_ptr(), ws_bytes=1 << 24, q_stride=256, B=1):
        return tb.lib.tb_kv4_attention_f32(out.data_ptr(), q.data_ptr(), q_stride, pages.data_ptr(), table.data_ptr(),
                                           lens.data_ptr(), starts.data_ptr(), None, B, 1, 1, H, 2, D, block, 2, 4,
                                           0.125, ws_ptr, ws_bytes, s)

    need = int(tb.lib.tb_kv4_attention_workspace_size(1, 4, 2, 64, 1))
    assert 0 < need <= 1 << 24
    assert attention(ws_bytes=need) == tb.TB_SUCCESS
    assert attention(ws_bytes=need - 1) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(ws_ptr=None) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(H=3) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(block=8) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(q_stride=255) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(D=48, q_stride=512) == tb.TB_ERROR_NOT_SUPPORTED
    assert attention(B=4096) == tb.TB_ERROR_NOT_SUPPORTED
    assert attention(B=-1) == tb.TB_ERROR_INVALID_ARGUMENT
    assert attention(block=1 << 26) == tb.TB_ERROR_NOT_SUPPORTED  # a page above 2 GB

    def append(T=1, Hkv=2, D=64, block=16, k_stride=128, cos=None, pos=None, pages_ptr=pages.data_ptr()):
        k = f32(4, 2, 64)
        return tb.lib.tb_kv4_append_rope_f32(pages_ptr, None, None, k.data_ptr(), k.data_ptr(), 0, k_stride, 128, cos,
                                             cos, pos, table.data_ptr(), None, T, 0, Hkv, D, block, 4, 9, s)

    assert append() == tb.TB_SUCCESS
    assert append(T=-1) == append(block=24) == append(k_stride=127) == tb.TB_ERROR_INVALID_ARGUMENT
    assert append(pages_ptr=pages.data_ptr() + 8) == tb.TB_ERROR_INVALID_ARGUMENT
    assert append(cos=ws.data_ptr()) == tb.TB_ERROR_INVALID_ARGUMENT  # no positions
    assert append(D=48) == tb.TB_ERROR_NOT_SUPPORTED
    with pytest.raises(tb.ShapeError):  # RoPE tables of another type
        be.KV4AppendRoPE(pages, f32(1, 2, 64), f32(1, 2, 64), f32(9, 32).half(), f32(9, 32).half(), i32(1), i32(1))

    def read(T=1, D=64, block=16, k=ws.data_ptr()):
        return tb.lib.tb_kv4_read_f32(k, ws.data_ptr() + 4096, pages.data_ptr(), table.data_ptr(), T, 2, D, block, 4, s)

    assert read() == tb.TB_SUCCESS
    assert read(T=-1) == read(block=8) == read(k=None) == tb.TB_ERROR_INVALID_ARGUMENT
    assert read(D=96) == tb.TB_ERROR_NOT_SUPPORTED

    def verify(B=1, K=2, V=8, row=8, p=ws.data_ptr()):
        tokens = torch.zeros(3, dtype=torch.int64, device=cuda)
        return tb.lib.tb_verify_draft_f32(tokens.data_ptr(), table.data_ptr(), p, 24, row, tokens.data_ptr(), None, 0,
                                          0, None, q.data_ptr(), None, B, K, V, s)

    assert verify() == tb.TB_SUCCESS
    assert verify(B=-1) == verify(K=-1) == verify(V=0) == verify(row=7) == verify(p=None) == \
        tb.TB_ERROR_INVALID_ARGUMENT
    assert verify(V=(1 << 26) + 1, row=1 << 27) == tb.TB_ERROR_NOT_SUPPORTED
    assert tb.lib.tb_kv4_tile_bytes(128) == 2176 and tb.lib.tb_kv4_tile_bytes(96) == 0
    c = i32(1)
    assert tb.lib.tb_kv4_plan(starts.data_ptr(), lens.data_ptr(), None, None, c.data_ptr(), None, table.data_ptr(),
                              i32(4).data_ptr(), c.data_ptr(), lens.data_ptr(), lens.data_ptr(), lens.data_ptr(), 1, 0,
                              2, 4, 16, s) == tb.TB_ERROR_INVALID_ARGUMENT  # count read and written in one word


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("entry", [-1, -2, -3, -2**31, 2**31 - 1])
def test_attention_no_value_of_an_entry_is_special(be, cuda, new, entry):
    """Whatever a bad entry's value, its page is hidden and counted once: the first and the second page of a
    32-position chunk, and the last one.  4, 8 and 160 query rows: each form of the kernels."""
    import torch

    rng = np.random.default_rng(30)
    n, D = 200, 64
    cache = Cache(be, rng, [n], 1, D, 16)
    hidden = [2, 5, 12]
    cache.table[0, hidden] = entry
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = rng.standard_normal((new, 4, D)).astype(np.float32)
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)),
                              _dev(np.array([0, new], np.int32)), new, bad=bad))
    for i in range(new):
        seen = np.arange(n - new + i + 1)
        seen = seen[~np.isin(seen // 16, hidden)]
        s = np.einsum("hd,jd->hj", q[i].astype(np.float64), cache.k[0][seen, 0]) / math.sqrt(D)
        p = np.exp(s - s.max(-1, keepdims=True))
        want = (p / p.sum(-1, keepdims=True)) @ cache.v[0][seen, 0]
        assert np.abs(got[i] - want).max() <= ATTN_TOL * np.abs(cache.v[0]).max(), i
    assert int(bad) == len(hidden)


def test_append_refuses_rope_tables_of_other_shapes(tb, be, cuda):
    """The tables' first dimension is the positions they reach: nothing but [max_seq, D / 2] is taken."""
    import torch

    D = 64
    pages, x = be.KV4Pages(1, 1, D, 16), torch.zeros(1, 1, D, device=cuda)
    i = torch.zeros(1, dtype=torch.int32, device=cuda)
    for shape in ((D // 2,), (1, 9, D // 2), (9, 1, D // 2), (9, D // 2 + 1), (9, D)):
        t = torch.zeros(*shape, device=cuda)
        with pytest.raises(tb.ShapeError):
            be.KV4AppendRoPE(pages, x, x, t, t, i, i)
    with pytest.raises(tb.ShapeError):
        be.KV4AppendRoPE(pages, x, x, torch.zeros(9, D // 2, device=cuda), torch.zeros(8, D // 2, device=cuda), i, i)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_rows_before_the_first_request_are_zero(tb, be, cuda, new):
    """Offsets that begin past the first row, as a later part of a batch has them: those rows are of no request."""
    import torch

    rng = np.random.default_rng(31)
    lens, news, lead, D = [90, 41], [new, new], 7, 64
    cache = Cache(be, rng, lens, 2, D, 16)
    q = rng.standard_normal((lead + 2 * new + 3, 8, D)).astype(np.float32)
    dq, out = _dev(q), torch.full(q.shape, float("nan"), device=cuda)
    table, lens32 = _dev(cache.table), _dev(np.array(lens, np.int32))
    starts = _dev((lead + np.array([0, new, 2 * new])).astype(np.int32))
    ws = torch.empty(int(tb.lib.tb_kv4_attention_workspace_size(len(q), 8, 2, D, new)), dtype=torch.uint8, device=cuda)
    tb.check(tb.lib.tb_kv4_attention_f32(
        out.data_ptr(), dq.data_ptr(), 8 * D, cache.pages.data_ptr(), table.data_ptr(), lens32.data_ptr(),
        starts.data_ptr(), None, 2, len(q), new, 8, 2, D, 16, cache.table.shape[1], cache.pages.shape[0], D**-0.5,
        ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    got = _np(out)
    want, most = attend_ref(cache, q[lead:lead + 2 * new], news, D**-0.5)
    assert (np.abs(got[lead:lead + 2 * new] - want).max((1, 2)) <= ATTN_TOL * most).all()
    assert (got[:lead] == 0).all() and (got[lead + 2 * new:] == 0).all()


def test_attention_prompts_far_apart_in_a_batch(be, cuda):
    """Two prompts with 1000 single tokens between them: right, and about as fast as side by side (where the
    order of the same requests costs nothing, it stays well below twice the time)."""
    import torch

    rng = np.random.default_rng(32)
    H, D, n = 33, 32, 1000  # the boundary between the prompts lies within a CTA's share
    best = {}
    for name, order in (("apart", [0] + list(range(2, n + 2)) + [1]), ("together", [0, 1] + list(range(2, n + 2)))):
        lens = np.where(np.arange(n + 2) < 2, 400, 1 + np.arange(n + 2) % 30)[order].tolist()
        news = np.where(np.arange(n + 2) < 2, 100, 1)[order].tolist()
        cache = Cache(be, rng, lens, H, D, 16)
        q = rng.standard_normal((sum(news), H, D)).astype(np.float32)
        _check_attention(be, cache, q, news)
        args = (_dev(q), cache.pages, _dev(cache.table), _dev(np.array(lens, np.int32)),
                _dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), 100)
        times = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            be.KV4Attention(*args)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        best[name] = min(times)
    assert best["apart"] < 2 * best["together"], best


def test_plan_from_several_threads(tb, cuda):
    """Plans of different sizes at the same time, a host thread each: none changes what another's launch may use."""
    import threading

    import torch

    sizes, status = (16384, 4000, 12000, 5000), {}
    work = []
    for B in sizes:  # empty requests: nothing but the launches counts
        zero = torch.zeros(B + 1, dtype=torch.int32, device=cuda)
        out = torch.zeros(2 * B + 64, dtype=torch.int32, device=cuda)
        at = lambda n: out.data_ptr() + 4 * n  # noqa: E731,B023
        args = (at(0), at(B + 8), None, None, at(2 * B + 16), at(2 * B + 17)) + (zero.data_ptr(),) * 6
        work.append((B, (zero, out), args + (B, 0, 1, 4, 16, torch.cuda.Stream().cuda_stream)))
    torch.cuda.synchronize()

    def call(B, args):
        status[B] = {tb.lib.tb_kv4_plan(*args) for _ in range(5000)}

    threads = [threading.Thread(target=call, args=(B, args)) for B, _, args in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == {B: {tb.TB_SUCCESS} for B in sizes}


WAITS = """
import json, sys
sys.path.insert(0, "tests")
import numpy as np, torch, tendo_b200 as tb
from test_gpu_kv4 import Cache, _dev, _np, attend_ref, ATTN_TOL
be, rng = tb.Backend(0), np.random.default_rng(37)
lens, news, D = [900, 300, 2000, 40, 700], [300, 129, 60, 40, 1], int(sys.argv[1])
cache = Cache(be, rng, lens, 2, D, 16)
q = rng.standard_normal((sum(news), 4, D)).astype(np.float32)
want, most = attend_ref(cache, q, news, D ** -0.5)
args = (_dev(q), cache.pages, _dev(cache.table), _dev(np.array(lens, np.int32)),
        _dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), 300)
for call in range(20):
    got = _np(be.KV4Attention(*args))
    err = np.abs(got - want) / most[:, None, None]
    assert (np.isnan(err) | (err <= ATTN_TOL)).all(), np.nanmax(err)
    try:
        be.KV4Check()
        assert np.isfinite(got).all()
        print("fine")
    except tb.TendoB200Error as e:
        assert e.code == tb.TB_ERROR_TIMEOUT and np.isnan(got).any()
        print("expired")
    be.KV4Check()  # said once
m = tb.QuantizedModel(json.load(open("tests/golden/tiny_greedy.json"))["config"], batch=1)
m.init_synthetic(0)
be.KV4Attention(*args)
print(m.generate_greedy(np.array([[1, 2]]), 2).shape)  # a model is not blamed for it
"""


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("polls", ["", "1", "2", "6"])
def test_waits_that_run_out_are_reported(cuda, D, polls):
    """With a wait's limit cut to a few polls a call ends all the same, its rows are right or NaN, and the check
    raises; with the limit as it is, nothing is reported."""
    import os
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", WAITS, str(D)], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, TENDO_B200_KV4_POLLS=polls),
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]
    said = r.stdout.split()
    assert len(said) == 22  # (1, 2)
    if polls == "":
        assert said[:20] == ["fine"] * 20
    if polls == "1":
        assert "expired" in said


def test_attention_of_lengths_at_the_end_of_32_bits(be, cuda):
    """A length that only a broken caller gives, in a table wide enough for it (every entry the same page): cut,
    where rounding it up to whole tiles would have passed 32 bits, and so what attention over that page gives.
    A warp adds up 28000 chunks in fp32, each sum off by 2^-24 of itself: 4e-3 with numerator and denominator.
    A CTA of the other kernel adds up 14 million positions, which bounds nothing but the result's size."""
    import torch

    rng = np.random.default_rng(38)
    cache = Cache(be, rng, [16], 1, 32, 16)
    page = int(cache.table[0, 0])
    cache.table = np.zeros((1, 1), np.int32)
    table = torch.full((1, (1 << 27) + 16), page, dtype=torch.int32, device=cuda)
    lens = _dev(np.array([2**31 - 1], np.int32))
    q = (0.3 * rng.standard_normal((16, 4, 32))).astype(np.float32)
    most = np.abs(cache.v[0]).max()
    got = _np(be.KV4Attention(_dev(q[:1]), cache.pages, table, lens, _dev(np.array([0, 1], np.int32)), 1))
    want, _ = attend_ref(cache, q[:1], [1], 1 / math.sqrt(32))
    assert np.abs(got - want).max() <= 4e-3 * most
    got = _np(be.KV4Attention(_dev(np.tile(q, (1, 2, 1))), cache.pages, table, lens, _dev(np.array([0, 16], np.int32)),
                              16))
    assert np.abs(got).max() <= 2 * most  # no NaN either
    be.KV4Check()


def test_attention_chunk_sums_over_a_long_context(be, cuda):
    """Equal terms, whose roundings do not cancel: one CTA takes all 131072 positions of a row, the first with a
    score 0.997 above the others' in log2 units.  Every value is 1.25, and so is the result.  A row's numerator and
    denominator are two sums each of 8192 parts of 8 terms: partial sums are half of the whole on average, so the
    sums are off by at most (8192 / 2 + 8) 2^-24 each."""
    import torch

    n, D, Hkv, G, new = 131072, 32, 37, 8, 128  # 148 units of 256 rows
    c = 0.5 + 0.98 * 2.0**-10  # in the second half of its sum every term loses nearly half a place
    pages, table = be.KV4Pages(n // 64, Hkv, D, 64), torch.arange(n // 64, dtype=torch.int32, device=cuda)[None]
    k, v = torch.zeros(n, Hkv, D, device=cuda), torch.full((n, Hkv, D), 1.25, device=cuda)
    k[0] = 1.0
    be.KV4AppendRoPE(pages, k, v, None, None, None, torch.arange(n, dtype=torch.int32, device=cuda))
    q = torch.full((new, Hkv * G, D), -math.log(c) / D, device=cuda)
    out = be.KV4Attention(q, pages, table, _dev(np.array([n], np.int32)), _dev(np.array([0, new], np.int32)), new, 1.0)
    assert np.abs(_np(out).astype(np.float64) / 1.25 - 1).max() <= 2 * (8192 / 2 + 8) * 2.0**-24


def test_append_of_values_at_the_end_of_fp32(be, cuda):
    """Up to 2^127 every row is held; past it a row without a finite scale reads back as NaN, as a whole."""
    D = 32
    big, most = np.float32(2.0**127), np.finfo(np.float32).max
    alternate = np.where(np.arange(D) % 2, 1, -1).astype(np.float32)
    v = np.stack([big * alternate, np.full(D, big), np.full(D, -big), most * alternate, np.full(D, most),
                  np.full(D, -most)])[:, None].astype(np.float32)
    pages, slots = be.KV4Pages(1, 1, D, 16), _dev(np.arange(len(v), dtype=np.int32))
    be.KV4AppendRoPE(pages, _dev(v), _dev(v), None, None, None, slots)
    for got in be.KV4Read(pages, slots):
        got = _np(got)
        u, scale, zero = quantize_rows(v[:3])
        np.testing.assert_array_equal(got[:3], values_of(u, scale, zero))
        assert (np.abs(got[:3].astype(np.float64) - v[:3]) <= 0.5 * scale[..., None] * (1 + 1e-5)).all()
        assert np.isnan(got[3:]).all()


@pytest.mark.parametrize("new", [1, 40])
def test_a_step_captured_once_and_replayed(be, cuda, new):
    """Plan, append, attention and verification in one graph: a replay with other lengths, rows and
    probabilities in the same buffers gives what the calls give, bit for bit."""
    import torch

    rng = np.random.default_rng(33)
    B, H, Hkv, D, bs, V, K = 3, 8, 2, 64, 16, 1000, 3
    T, NB = B * new, 64
    cos, sin = (_dev(t) for t in be.RoPETables(D, 512, 10000.0))
    names = ("held", "ctx", "new", "table", "free", "count", "rows", "p", "x", "u")
    state = {}

    def fresh(ctx, news):
        have = [_up(c, bs) for c in ctx]
        table = np.full((B, 20), -1, np.int32)
        order = rng.permutation(NB).astype(np.int32)
        for b in range(B):
            table[b, :have[b]] = order[sum(have[:b]):sum(have[:b + 1])]
        free = np.zeros(NB, np.int32)
        free[:NB - sum(have)] = order[sum(have):]
        p = _probs(rng, B, K + 1, V)
        return dict(held=np.array(ctx, np.int32), ctx=np.array(ctx, np.int32), new=np.array(news, np.int32), table=table,
                    free=free, count=np.array([NB - sum(have)], np.int32), rows=_rows(rng, T, H + 2 * Hkv, D), p=p,
                    x=p[:, :K].argmax(-1), u=rng.random((B, K + 1)).astype(np.float32) * np.float32(0.5))

    pages = be.KV4Pages(NB, Hkv, D, bs)

    def step():
        s = state
        plan = be.KV4Plan(s["held"], s["ctx"], s["new"], s["table"], s["free"], s["count"], T, bs)
        r = s["rows"]
        q = be.KV4AppendRoPE(pages, r[:, H:H + Hkv], r[:, H + Hkv:], cos, sin, plan.positions, plan.slots, q=r[:, :H])
        out = be.KV4Attention(q, pages, s["table"], plan.seq_lens, plan.q_start, new)
        return (out, plan.slots, plan.free_count) + be.VerifyDraft(s["p"], s["x"], s["u"])

    def load(values):
        for name in names:
            if name in state:
                state[name].copy_(_dev(values[name]))
            else:
                state[name] = _dev(values[name])

    content = torch.from_numpy(rng.integers(0, 256, tuple(pages.shape), np.uint8))
    content[..., 16 * D:] = 0
    first = fresh([100, 37, 5], [new, new, new])
    load(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for values in (first, fresh([200, 0, 63], [new, new - 1, new]), fresh([15, 16, 17], [0, 1, new])):
        results = []
        for replay in (False, True):
            load(values)
            pages.copy_(content)
            if replay:
                graph.replay()
                results.append([t.clone() for t in held] + [pages.clone(), state["table"].clone()])
            else:
                results.append([t.clone() for t in step()] + [pages.clone(), state["table"].clone()])
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_the_first_call_of_a_process_may_be_captured(cuda):
    """Nothing that a first call sets up (function attributes, addresses of device words) breaks a capture."""
    import os
    import subprocess
    import sys

    code = (
        "import sys; sys.path.insert(0, 'tests'); import numpy as np, torch, tendo_b200 as tb\n"
        "be = tb.Backend(0)\n"
        "i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device='cuda')\n"
        "pages, x = be.KV4Pages(8, 1, 64, 16), torch.ones(90, 3, 64, device='cuda')\n"
        "held, new, table, free, count = i32(1), i32(1) + 90, i32(1, 8), torch.arange(8, device='cuda').int(), i32(1) + 8\n"
        "p, d, u = torch.full((1, 2, 9), 1 / 9, device='cuda'), i32(1, 1).long(), torch.zeros(1, 2, device='cuda')\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    s = be.KV4Plan(held, held, new, table, free, count, 90, 16)\n"
        "    q = be.KV4AppendRoPE(pages, x[:, 1:2], x[:, 2:], None, None, None, s.slots, q=x[:, :1])\n"
        "    o = be.KV4Attention(q, pages, table, s.seq_lens, s.q_start, 90)\n"
        "    o1 = be.KV4Attention(q, pages, table, s.seq_lens, s.q_start, 1)\n"
        "    t, a = be.VerifyDraft(p, d, u)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "print(int(s.bad), bool(torch.isfinite(o).all()), float((o - 1).abs().max()) < 1e-5,\n"
        "      float((o1 - 1).abs().max()) < 1e-5, int(a))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["0", "True", "True", "True", "1"], r.stdout


@pytest.mark.parametrize("new", [1, 9])
def test_attention_of_a_long_context(be, cuda, new):
    """150001 positions, 1 and 72 rows a kv head: offsets and counts of a long document in both kernels."""
    rng = np.random.default_rng(34)
    lens = [150001, 40]
    cache = Cache(be, rng, lens, 1, 64, 64)
    q = rng.standard_normal((2 * new, 8, 64)).astype(np.float32)
    _check_attention(be, cache, q, [new, new])


def test_attention_past_32_bits_of_cache(be, cuda):
    """Pages that lie past 4 GB of the cache, as a table's order may have them."""
    import torch

    rng = np.random.default_rng(35)
    Hkv, D, block, n = 8, 128, 64, 500
    lens = [n, 70]
    cache = Cache(be, rng, lens, Hkv, D, block)
    NB = (5 << 30) // (Hkv * (block // 16) * (16 * D + 128))
    big = torch.empty(NB, *cache.pages.shape[1:], dtype=torch.uint8, device=cuda)
    shift = NB - cache.pages.shape[0]
    big[shift:] = cache.pages
    cache.pages, cache.table = big, np.where(cache.table >= 0, cache.table + shift, cache.table).astype(np.int32)
    for news in ([1, 1], [60, 70]):
        q = rng.standard_normal((sum(news), 16, D)).astype(np.float32)
        _check_attention(be, cache, q, news)
    slots = _dev((cache.table[0, np.arange(n) // block] * block + np.arange(n) % block).astype(np.int32))
    k, v = be.KV4Read(cache.pages, slots)
    np.testing.assert_array_equal(_np(k), cache.k[0].astype(np.float32))
    np.testing.assert_array_equal(_np(v), cache.v[0].astype(np.float32))
    x = _rows(rng, n, Hkv, D)
    be.KV4AppendRoPE(cache.pages, _dev(x), _dev(x), None, None, None, slots)
    np.testing.assert_array_equal(_np(be.KV4Read(cache.pages, slots)[0]), values_of(*quantize_rows(x)))


def test_plan_of_the_most_requests(be, cuda):
    """B = 16384, the largest that is taken; one more is refused."""
    import torch

    import tendo_b200 as tb

    rng = np.random.default_rng(36)
    B, bs = 16384, 16
    held = rng.integers(0, 40, B)
    ctx = np.where(rng.random(B) < 0.3, held // 2, held)
    new = rng.integers(0, 20, B)
    table, free, count = _plan_state(rng, held.tolist(), bs, 6, int(sum(_up(c + n, bs) for c, n in zip(ctx, new))))
    want = _check_plan(be, held.tolist(), ctx.tolist(), new.tolist(), table, free, count, int(new.sum()) + 1, bs)
    assert want[-1] == 0
    z = torch.zeros(B + 1, dtype=torch.int32, device=cuda)
    with pytest.raises(tb.TendoB200Error) as e:
        be.KV4Plan(z, z, z, torch.zeros(B + 1, 1, dtype=torch.int32, device=cuda), z[:4].clone(), z[:1].clone(), 1, bs)
    assert e.value.code == tb.TB_ERROR_NOT_SUPPORTED


@pytest.mark.parametrize("H,Hkv,D", [(200, 1, 32), (1000, 2, 64), (129, 1, 128)])
@pytest.mark.parametrize("new", [1, 7])
def test_attention_of_large_groups(be, cuda, H, Hkv, D, new):
    """More heads to a kv head than the kernel for many rows takes."""
    rng = np.random.default_rng(39)
    lens = [1, 70, 300]
    news = [min(new, n) for n in lens]
    cache = Cache(be, rng, lens, Hkv, D, 16)
    _check_attention(be, cache, rng.standard_normal((sum(news), H, D)).astype(np.float32), news)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("k", [0, 8, 14, 20])
def test_attention_beside_a_far_larger_value(be, cuda, new, k):
    """One position whose values are 2^k times the others' and whose score leaves it no weight.  V's scales share
    a power of two that brings the largest to 2^6 .. 2^7, in fp16 terms down to 2^-24: the others' products with p
    are off by 2^-25 of 2^(6 - k) at most, 2^(k - 31) of the result, beside the tolerance of any attention."""
    rng = np.random.default_rng(40 + k)
    n, D, at = 300, 32, 137  # not the first position that a warp or a tile meets
    cache = Cache(be, rng, [n], 1, D, 16)
    key, v = np.zeros((n, 1, D), np.float32), rng.standard_normal((n, 1, D)).astype(np.float32)
    key[at], v[at] = -40.0, np.ldexp(v[at], k)
    slots = (cache.table[0, np.arange(n) // 16] * 16 + np.arange(n) % 16).astype(np.int32)
    be.KV4AppendRoPE(cache.pages, _dev(key), _dev(v), None, None, None, _dev(slots))
    cache.k[0], cache.v[0] = (values_of(*quantize_rows(x)).astype(np.float64) for x in (key, v))
    q = np.ones((new, 4, D), np.float32)
    got = _np(be.KV4Attention(_dev(q), cache.pages, _dev(cache.table), _dev(np.array([n], np.int32)),
                              _dev(np.array([0, new], np.int32)), new))
    want, _ = attend_ref(cache, q, [new], 1 / math.sqrt(D))
    small = np.abs(np.delete(cache.v[0], at, 0)).max()
    assert np.abs(got - want).max() <= (ATTN_TOL + 2.0 ** (k - 31)) * small
