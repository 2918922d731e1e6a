"""The operators of paged serving over a 4-bit KV cache: what is measured.

Four operators, used in this order by a serving step with drafted tokens:
  plan    block tables and slot maps on the GPU from request lengths
  append  RoPE on q and k, K and V rows to 4 bits into their pages, and the rows read back
  attend  attention over the paged 4-bit cache: single tokens, drafted tokens, prompt chunks
  verify  drafted tokens against the target's probabilities, from given random numbers

With ``own`` false ``run`` computes them from elementary torch operations, with
``own`` true through tendo_b200's entry points.  Head counts are those of the
7B (32 heads) and 70B (64 heads on 8 kv heads) shapes this repository serves.

A cache tile holds 16 positions of one kv head: K codes [16][D/2], V codes
[16][D/2] (two 4-bit codes to a byte, the even channel low, code + 8), then
for K and for V one 32-bit word per position, bf16 scale low, bf16 zero high;
value = zero + scale * code, codes -8 .. 7.
"""
import math
import random

import torch

own = False

_DEV = "cuda"
_backend = None


def _be():
    global _backend
    if _backend is None:
        import tendo_b200

        _backend = tendo_b200.Backend(torch.cuda.current_device())
    return _backend


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the step of a 64-request server: every request adds one token, a few finish or roll back
        dict(name="plan decode 64", op="plan", requests=64, ctx=1024, new=1, block=16, columns=256),
        # admission with prompt chunks: 1024 requests, some of them hundreds of new tokens
        dict(name="plan mixed 1024", op="plan", requests=1024, ctx=700, new=61, block=32, columns=128),
        # one decode step's rows of a 7B layer, 64 sequences
        dict(name="append 7B 64 tokens", op="append", tokens=64, heads=32, kv_heads=32, dim=128, block=16),
        # a prompt's rows of a 70B layer
        dict(name="append 70B prompt", op="append", tokens=8192, heads=64, kv_heads=8, dim=128, block=16),
        # one user, one token: latency
        dict(name="attend 7B one", op="attend", requests=1, ctx=601, new=1, heads=32, kv_heads=32, dim=128, block=16),
        # serving decode, 64 ragged sequences, a kv head for each head
        dict(name="attend 7B serving", op="attend", requests=64, ctx=1500, new=1, heads=32, kv_heads=32, dim=128,
             block=16),
        # decode of the 70B shape, grouped heads
        dict(name="attend 70B serving", op="attend", requests=16, ctx=2100, new=1, heads=64, kv_heads=8, dim=128,
             block=16),
        # the same with four drafted tokens each
        dict(name="attend 70B drafts", op="attend", requests=16, ctx=2100, new=5, heads=64, kv_heads=8, dim=128,
             block=32),
        # one long document
        dict(name="attend 70B long", op="attend", requests=1, ctx=131011, new=1, heads=64, kv_heads=8, dim=128,
             block=64),
        # prompt chunks over what came before
        dict(name="attend 70B prompt", op="attend", requests=4, ctx=2000, new=1000, heads=64, kv_heads=8, dim=128,
             block=16),
        # one request, four drafts, the vocabulary of the 7B shape
        dict(name="verify one", op="verify", requests=1, drafts=4, vocab=32000),
        # a batch at a large vocabulary
        dict(name="verify 64", op="verify", requests=64, drafts=7, vocab=128000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1e15)


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "verify"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        block = rng.choice([16, 32, 64, 128])
        if op == "plan":
            ctx, new = _log(rng, 1, 4000), _log(rng, 1, 300)
            c = dict(op=op, requests=_log(rng, 1, 1500), ctx=ctx, new=new, block=block,
                     columns=(5 * (ctx + new) + 40) // block + 2)
        elif op == "verify":
            c = dict(op=op, requests=_log(rng, 1, 64), drafts=rng.randint(1, 8), vocab=_log(rng, 1000, 128000))
        else:
            dim = rng.choice([32, 64, 128, 128])
            kv = rng.choice([1, 2, 4, 8, 8, 32])
            group = rng.choice([1, 2, 3, 4, 6, 8]) if kv < 32 else 1
            if op == "append":
                c = dict(op=op, tokens=_log(rng, 1, 8192), heads=kv * group, kv_heads=kv, dim=dim, block=block)
            else:
                new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 1000)])
                ctx = _log(rng, 1, 131072) if rng.random() < 0.3 else _log(rng, 1, 4096)
                c = dict(op=op, requests=_log(rng, 1, 64), ctx=ctx, new=new, heads=kv * group, kv_heads=kv, dim=dim,
                         block=block)
                longest = max(a + b for a, b in zip(*_lengths(c)))
                if c["requests"] * c["heads"] * max(_lengths(c)[1]) * longest > 1.5e9:
                    continue  # the plain form holds every score at once
                if c["requests"] * c["kv_heads"] * longest * dim > 1.2e9:
                    continue
        if _cost(c) <= most:
            return c


def _lengths(case):
    """Per request (tokens in the cache before the call, new tokens), spread around the case's figures.

    Serving is ragged: contexts lie between 0.5 and 1.5 of ``ctx``; single tokens and drafts are the same for
    every request, chunks of more than 16 lie between half and the whole."""
    r = random.Random("%s %s %s" % (case["requests"], case["ctx"], case["new"]))
    n = case["requests"]
    if n == 1:
        return [case["ctx"]], [case["new"]]
    ctx = [int(case["ctx"] * r.uniform(0.5, 1.5)) for _ in range(n)]
    new = [case["new"] if case["new"] <= 16 else r.randint((case["new"] + 1) // 2, case["new"]) for _ in range(n)]
    return ctx, new


def _plan_lengths(case):
    """(held, ctx, new) per request: most go on, one in eight rolled back drafts, one in sixteen finished,
    one in sixteen is new; those that add a prompt chunk add up to eight times ``new``."""
    r = random.Random("plan %s %s %s" % (case["requests"], case["ctx"], case["new"]))
    held, ctx, new = [], [], []
    for _ in range(case["requests"]):
        c = int(case["ctx"] * r.uniform(0.5, 1.5))
        n = case["new"] if case["new"] <= 8 else int(case["new"] * math.exp(r.uniform(-2, 1.5)))
        h = c
        what = r.randrange(16)
        if what == 0:
            c, n = 0, 0
        elif what == 1:
            h = c = 0
            n = max(n, min(case["ctx"], 4 * n))
        elif what in (2, 3):
            h = c + r.randint(1, 40)
        held.append(h)
        ctx.append(c)
        new.append(n)
    return held, ctx, new


def _blocks(n, size):
    return (n + size - 1) // size


def work(case):
    op = case["op"]
    if op == "plan":
        held, ctx, new = _plan_lengths(case)
        moved = sum(abs(_blocks(c + n, case["block"]) - _blocks(h, case["block"])) for h, c, n in zip(held, ctx, new))
        # lengths in, sequence lengths and token offsets out; each page moved read and written; position and slot out
        return {"bytes": 20.0 * len(ctx) + 8.0 * moved + 8.0 * sum(new), "flops": 4.0 * (sum(new) + moved)}
    if op == "append":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        rows = t * kv * 2
        # fused rows in, rotated q and packed rows out; then packed rows in and values out
        return {"bytes": 4.0 * t * (h + 2 * kv) * d + 4.0 * t * h * d + 2.0 * rows * (d // 2 + 4) + 4.0 * rows * d,
                "flops": 3.0 * t * (h + kv) * d + 8.0 * rows * d}
    if op == "attend":
        ctx, new = _lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        keys = sum(c + n for c, n in zip(ctx, new))
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
        return {"bytes": float(keys * kv * (d + 8) + 8 * sum(new) * h * d), "flops": 4.0 * d * h * pairs}
    b, v = case["requests"], case["vocab"]
    return {"bytes": 8.0 * b * v, "flops": 4.0 * b * v}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "plan":
        return _prepare_plan(case, g)
    if op == "append":
        return _prepare_append(case, g)
    if op == "attend":
        return _prepare_attend(case, g)
    b, k, v = case["requests"], case["drafts"], case["vocab"]
    # the drafter's logits are the target's with an error, as a small model's are
    target = torch.empty(b, k + 1, v, device=_DEV).normal_(0, 3.0, generator=g)
    draft = target[:, :k] + torch.empty(b, k, v, device=_DEV).normal_(0, 0.8, generator=g)
    p, q = torch.softmax(target, -1), torch.softmax(draft, -1)
    tokens = torch.multinomial(q.reshape(b * k, v), 1, generator=g).reshape(b, k)
    lens = torch.randint(max(0, k - 2), k + 1, (b,), generator=g, device=_DEV, dtype=torch.int32)
    u = torch.rand(b, k + 1, generator=g, device=_DEV)
    return dict(op=op, p=p, q=q, tokens=tokens, lens=lens, u=u)


def _prepare_plan(case, g):
    held, ctx, new = _plan_lengths(case)
    bs, cols, n = case["block"], case["columns"], case["requests"]
    have = [_blocks(h, bs) for h in held]
    need = sum(_blocks(c + m, bs) for c, m in zip(ctx, new))
    total = sum(have) + need + 64
    order = torch.randperm(total, generator=g, device=_DEV).to(torch.int32)
    table = torch.full((n, cols), -1, dtype=torch.int32, device=_DEV)
    start = torch.tensor([sum(have[:i]) for i in range(n)] if n < 64 else _running(have), device=_DEV)
    col = torch.arange(cols, device=_DEV)
    held_here = col[None] < torch.tensor(have, device=_DEV)[:, None]
    table = torch.where(held_here, order[(start[:, None] + col[None]).clamp(max=total - 1)], table)
    free = torch.full((total,), -1, dtype=torch.int32, device=_DEV)
    used = sum(have)
    free[: total - used] = order[used:]
    tokens = sum(new) + 3  # a captured step keeps a few rows of padding
    return dict(op="plan", held=_i32(held), ctx=_i32(ctx), new=_i32(new), table=table, free=free,
                count=_i32([total - used]), tokens=tokens, block=bs)


def _running(values):
    out, s = [], 0
    for v in values:
        out.append(s)
        s += v
    return out


def _rope_tables(rows, dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=_DEV, dtype=torch.float64) / dim)
    a = torch.arange(rows, device=_DEV, dtype=torch.float64)[:, None] * inv[None]
    return a.cos().float(), a.sin().float()


def _prepare_append(case, g):
    t, h, kv, d, bs = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    qkv = torch.empty(t, (h + 2 * kv) * d, device=_DEV).normal_(0, 1, generator=g)
    # some key channels are much larger than the others in every trained model
    loud = 1 + 6 * (torch.rand(kv * d, generator=g, device=_DEV) < 0.03).float()
    qkv[:, h * d:(h + kv) * d] *= loud
    blocks = _blocks(t, bs) + 3
    pages = torch.zeros(blocks, kv, bs // 16, 16 * d + 128, dtype=torch.uint8, device=_DEV)
    first = int(torch.randint(0, 1000, (1,), generator=g, device=_DEV))
    cos, sin = _rope_tables(t + 1000, d)
    where = torch.randperm(blocks, generator=g, device=_DEV).to(torch.int32)
    i = torch.arange(t, device=_DEV, dtype=torch.int32)
    slots = where[(i // bs).long()] * bs + i % bs
    view = qkv.view(t, h + 2 * kv, d)
    return dict(op="append", q=view[:, :h], k=view[:, h:h + kv], v=view[:, h + kv:], cos=cos, sin=sin,
                positions=i + first, slots=slots, pages=pages)


def _prepare_attend(case, g):
    ctx, new = _lengths(case)
    h, kv, d, bs, n = case["heads"], case["kv_heads"], case["dim"], case["block"], case["requests"]
    lens = [c + m for c, m in zip(ctx, new)]
    have = [_blocks(x, bs) for x in lens]
    blocks = sum(have) + 2
    cols = max(have) + 3
    pages = torch.empty(blocks, kv, bs // 16, 16 * d + 128, dtype=torch.uint8, device=_DEV)
    loud = 1 + 4 * (torch.rand(kv, 1, 1, d, generator=g, device=_DEV) < 0.03).float()
    step = max(1, (1 << 26) // (kv * bs * d))
    for a in range(0, blocks, step):
        m = min(step, blocks - a)
        shape = (m, kv, bs // 16, 16, d)
        for part, amp in ((0, loud), (1, 1.0)):
            x = torch.empty(shape, device=_DEV).normal_(0, 1, generator=g) * amp
            codes, words = _quantize_rows(x)
            dst = pages[a:a + m]
            dst[..., part * 8 * d:(part + 1) * 8 * d] = codes.reshape(m, kv, bs // 16, 8 * d)
            dst[..., 16 * d + 64 * part:16 * d + 64 * part + 64] = words.view(torch.uint8).reshape(m, kv, bs // 16, 64)
    order = torch.randperm(blocks, generator=g, device=_DEV).to(torch.int32)
    col = torch.arange(cols, device=_DEV)
    start = torch.tensor(_running(have), device=_DEV)
    table = torch.where(col[None] < torch.tensor(have, device=_DEV)[:, None],
                        order[(start[:, None] + col[None]).clamp(max=blocks - 1)], -1)
    t = sum(new)
    q = torch.empty(t, h, d, device=_DEV).normal_(0, 1.5, generator=g)
    return dict(op="attend", q=q, pages=pages, table=table.to(torch.int32), lens=_i32(lens),
                starts=_i32(_running(new) + [t]), most=max(new), longest=max(lens), scale=1.0 / math.sqrt(d))


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def _own(s):
    be = _be()
    if s["op"] == "plan":
        p = be.KV4Plan(s["held"], s["ctx"], s["new"], s["table"], s["free"], s["count"], s["tokens"], s["block"])
        return dict(table=s["table"], free=s["free"], count=p.free_count, lens=p.seq_lens, starts=p.q_start,
                    positions=p.positions, slots=p.slots)
    if s["op"] == "append":
        q = be.KV4AppendRoPE(s["pages"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], q=s["q"])
        k, v = be.KV4Read(s["pages"], s["slots"])
        return dict(q=q, k=k, v=v)
    if s["op"] == "attend":
        return be.KV4Attention(s["q"], s["pages"], s["table"], s["lens"], s["starts"], s["most"], s["scale"])
    tokens, accepted = be.VerifyDraft(s["p"], s["tokens"], s["u"], draft_probs=s["q"], draft_lens=s["lens"])
    return dict(tokens=tokens, accepted=accepted)


def _plain_plan(s):
    held, ctx, new, table, free, bs = s["held"], s["ctx"], s["new"], s["table"], s["free"], s["block"]
    n, cols = table.shape
    have, need = (held + bs - 1) // bs, (ctx + new + bs - 1) // bs
    give, take = (have - need).clamp(min=0), (need - have).clamp(min=0)
    give_end, take_end = give.cumsum(0), take.cumsum(0)
    top = s["count"] + give_end[-1:]
    col = torch.arange(cols, device=table.device, dtype=torch.int32)[None]
    # surplus pages on the stack in request order, then the missing ones off it in request order
    pushed = (col >= need[:, None]) & (col < have[:, None])
    at = s["count"] + (give_end - give)[:, None] + col - need[:, None]
    stack = torch.cat([free, free[:1]])
    stack = stack.scatter(0, torch.where(pushed, at, free.numel()).reshape(-1).long(), table.reshape(-1))[:-1]
    popped = (col >= have[:, None]) & (col < need[:, None])
    at = top - 1 - ((take_end - take)[:, None] + col - have[:, None])
    table = torch.where(popped, stack[at.clamp(0, free.numel() - 1).long()], table)
    ends = new.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    t = torch.arange(s["tokens"], device=table.device, dtype=torch.int64)
    b = torch.searchsorted(ends, t, right=True)
    real = b < n
    b = b.clamp(max=n - 1)
    pos = torch.where(real, ctx[b] + t - starts[b], 0)
    slots = torch.where(real, table[b, pos // bs].long() * bs + pos % bs, -1)
    return dict(table=table, free=stack, count=(top - take_end[-1:]).to(torch.int32), lens=ctx + new, starts=starts,
                positions=pos.to(torch.int32), slots=slots.to(torch.int32))


def _bf16_up(x):
    """The smallest bf16 value not below x (x >= 0 and finite), as fp32."""
    return ((x.contiguous().view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)


def _quantize_rows(x):
    """Rows of the last dimension as (codes uint8 [..., D/2], words int32 [...])."""
    mn, mx = x.amin(-1), x.amax(-1)
    zero = (mn * (7 / 15) + mx * (8 / 15)).to(torch.bfloat16).float()
    scale = _bf16_up(torch.maximum((zero - mn) * 0.125, (mx - zero) * (1 / 7)))
    c = torch.round((x - zero[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None])
    u = torch.where(scale[..., None] > 0, c.clamp(-8, 7), 0.0).to(torch.int32) + 8
    codes = (u[..., 0::2] | (u[..., 1::2] << 4)).to(torch.uint8)
    words = zero.view(torch.int32) | ((scale.view(torch.int32) >> 16) & 0xFFFF)
    return codes, words


def _rows_of(pages, part):
    """Views of the code rows and of the words' bytes of K (part 0) or V (part 1)."""
    d = (pages.shape[-1] - 128) // 16
    codes = pages[..., part * 8 * d:(part + 1) * 8 * d].unflatten(-1, (16, d // 2))
    words = pages[..., 16 * d + 64 * part:16 * d + 64 * part + 64].unflatten(-1, (16, 4))
    return codes, words


def _values(codes, words):
    """fp32 values of code rows [..., D/2] with their words' bytes [..., 4]."""
    w = words.contiguous().view(torch.int32).squeeze(-1)
    scale, zero = (w << 16).view(torch.float32), (w & -65536).view(torch.float32)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    return zero[..., None] + scale[..., None] * c


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    pages, slots = s["pages"], s["slots"].long()
    bs = pages.shape[2] * 16
    blk, tile, row = slots // bs, slots % bs // 16, slots % 16
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    out = dict(q=_rotate(s["q"], cos, sin))
    for name, part, x in (("k", 0, _rotate(s["k"], cos, sin)), ("v", 1, s["v"])):
        codes, words = _quantize_rows(x)
        held_codes, held_words = _rows_of(pages, part)
        held_codes[blk, :, tile, row] = codes
        held_words[blk, :, tile, row] = words.view(torch.uint8).unflatten(-1, (-1, 4))
        out[name] = _values(held_codes[blk, :, tile, row], held_words[blk, :, tile, row])
    return out


def _plain_attend(s):
    pages, q = s["pages"], s["q"]
    blocks, kv, sub, _ = pages.shape
    t, h, d = q.shape
    n, most, bs = s["lens"].numel(), s["most"], sub * 16
    used = _blocks(s["longest"], bs)
    at = s["table"][:, :used].clamp(min=0).long()
    keys, vals = (_values(*_rows_of(pages[at], part)).transpose(1, 2).reshape(n, kv, used * bs, d) for part in (0, 1))
    start, count = s["starts"][:-1], s["starts"][1:] - s["starts"][:-1]
    i = torch.arange(most, device=q.device)
    rows = (start[:, None] + i[None]).clamp(max=t - 1).long()
    x = q[rows].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    scores = (x * s["scale"]) @ keys.transpose(-1, -2)
    scores = scores.view(n, kv, h // kv, most, used * bs)
    last = (s["lens"] - count)[:, None] + i[None]
    seen = torch.arange(used * bs, device=q.device)[None, None] <= last[..., None]
    seen &= (torch.arange(used * bs, device=q.device)[None] < s["lens"][:, None])[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p.view(n, kv, -1, used * bs) @ vals
    o = o.view(n, kv, h // kv, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, h, d)
    # back to the ragged rows
    token = torch.arange(t, device=q.device)
    b = torch.searchsorted(s["starts"][1:].long(), token, right=True)
    return o[b, token - start[b]]


def _draw(weights, u):
    """First index whose running sum of floor(w 2^36) exceeds floor(u S), per row."""
    w = (weights.clamp(max=1.0) * float(1 << 36)).to(torch.int64)
    ends = w.cumsum(-1)
    total = ends[:, -1]
    m = (u * float(1 << 24)).to(torch.int64)
    target = (total >> 24) * m + (((total & 0xFFFFFF) * m) >> 24)
    return torch.searchsorted(ends, target[:, None], right=True)[:, 0], total


def _plain_verify(s):
    p, q, x, lens, u = s["p"], s["q"], s["tokens"], s["lens"].long(), s["u"]
    b, k = x.shape
    px = p[:, :k].gather(2, x[..., None])[..., 0]
    qx = q.gather(2, x[..., None])[..., 0]
    i = torch.arange(k, device=x.device)[None]
    fine = (u[:, :k] * qx < px) & (i < lens[:, None])
    accepted = fine.to(torch.int64).cumprod(1).sum(1)
    row = torch.arange(b, device=x.device)
    target = p[row, accepted]
    refused = accepted < lens
    rest = target - torch.where(refused[:, None], q[row, accepted.clamp(max=k - 1)], 0.0)
    token, total = _draw(rest.clamp(min=0.0), u[:, k])
    again, _ = _draw(target, u[:, k])
    token = torch.where(total > 0, token, again)
    j = torch.arange(k + 1, device=x.device)[None]
    drafts = torch.cat([x, x[:, :1]], 1)
    tokens = torch.where(j < accepted[:, None], drafts, torch.where(j == accepted[:, None], token[:, None], -1))
    return dict(tokens=tokens, accepted=accepted.to(torch.int32))


_PLAIN = dict(plan=_plain_plan, append=_plain_append, attend=_plain_attend, verify=_plain_verify)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op in ("plan", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_append(s) if op == "append" else _exact_attend(s)


def _exact_append(s):
    at = s["positions"].long()
    d = s["q"].shape[-1]
    cos, sin = (s[n].double().index_select(0, at).unsqueeze(1) for n in ("cos", "sin"))

    def turned(x):
        lo, hi = x[..., : d // 2].double(), x[..., d // 2:].double()
        y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        y[..., : d // 2] = lo * cos - hi * sin
        y[..., d // 2:] = lo * sin + hi * cos
        return y

    def held(x):
        lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        zero = ((7 * lo + 8 * hi) / 15).bfloat16().double()
        want = torch.max((zero - lo) / 8, (hi - zero) / 7)
        near = want.bfloat16().double()
        step = torch.where(near < want, torch.ldexp(torch.ones_like(near), torch.frexp(near).exponent - 8), 0.0)
        scale = near + step
        return zero + scale * ((x - zero) / scale).round().clamp(-8, 7)

    return dict(q=turned(s["q"]), k=held(turned(s["k"])), v=held(s["v"].double()))


def _exact_attend(s):
    q, pages, scale = s["q"], s["pages"], s["scale"]
    _, kv, sub, size = pages.shape
    t, h, d = q.shape
    out = torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    group = h // kv
    for b, length in enumerate(lens):
        a, e = starts[b], starts[b + 1]
        mine = s["table"][b, : _blocks(length, sub * 16)].long()
        for head in range(kv):
            tiles = pages[mine, head].reshape(-1, size)
            rows = []
            for part in (0, 1):
                raw = tiles[:, part * 8 * d:(part + 1) * 8 * d].reshape(-1, d // 2)
                c = torch.empty(raw.shape[0], d, dtype=torch.float64, device=q.device)
                c[:, 0::2] = (raw % 16).double() - 8
                c[:, 1::2] = (raw // 16).double() - 8
                w = tiles[:, 16 * d + 64 * part:16 * d + 64 * part + 64].contiguous().view(torch.bfloat16)
                w = w.reshape(-1, 2).double()
                rows.append((c * w[:, :1] + w[:, 1:])[:length])
            for i in range(a, e, 256):  # a bounded block of queries
                n = min(256, e - i)
                x = q[i:i + n, head * group:(head + 1) * group].double().transpose(0, 1)
                z = torch.matmul(x, rows[0].T) * scale
                sees = torch.arange(length, device=q.device)[None] <= (length - (e - i)) + torch.arange(n, device=q.device)[:, None]
                z = torch.where(sees[None], z, -torch.inf)
                w = torch.softmax(z, -1)
                out[i:i + n, head * group:(head + 1) * group] = torch.matmul(w, rows[1]).transpose(0, 1)
    return out
