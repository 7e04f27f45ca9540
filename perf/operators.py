"""Attention over a key/value cache held in 4 bits: what is timed of it, in plain torch and through the library.

Four operators work on one paged cache.  `append` puts new keys and values into it (bias, rotary position, 4-bit rows; `read`
gives rows back as numbers), `attend` is attention over it for single tokens and for chunks of a prompt, `weights` adds up how
much attention every cached position got, and `evict` keeps the positions that got most and moves them to fresh pages.

A cached row (one position of one key/value head, 128 values) is quantised like a group of the library's weights, with a zero
point: value = (code - 8) * scale + zero, scale = fp16((max - min) / 15), zero = fp16(min + 8 scale).  A page record holds
`page` rows of one head: 16 words of codes per key row, the same for the value rows, then (scale, zero) per key row and per value
row, so 34 words per position.  A word is packed as the library's weight words are.
"""
import math
from types import SimpleNamespace

import torch

own = False

D = 128                                             # values of a head
SHIFTS = (0, 8, 16, 24, 4, 12, 20, 28)              # bit of element j of a packed word
ROPE_THETA = 1e6


def listed():
    return [
        # one new token of one short conversation: the latency of a decode step
        {"name": "append_token", "op": "append", "seqs": 1, "longest": 1000, "tokens": 1, "q_heads": 12, "kv_heads": 2, "page": 16},
        # four prompts of different lengths going in at once
        {"name": "append_prompts", "op": "append", "seqs": 4, "longest": 4100, "tokens": 4100, "q_heads": 12, "kv_heads": 2, "page": 64},
        # decode step of one conversation, short and very long; heads in fp32 as the O projection takes them
        {"name": "attend_token_short", "op": "attend", "seqs": 1, "longest": 1021, "tokens": 1, "q_heads": 12, "kv_heads": 2, "page": 16, "fp32": True},
        {"name": "attend_token_long", "op": "attend", "seqs": 1, "longest": 131001, "tokens": 1, "q_heads": 12, "kv_heads": 2, "page": 64, "fp32": True},
        # decode step of a large ragged batch
        {"name": "attend_batch", "op": "attend", "seqs": 64, "longest": 8190, "tokens": 1, "q_heads": 32, "kv_heads": 8, "page": 16, "fp32": False},
        # a few guessed tokens per sequence checked at once
        {"name": "attend_guesses", "op": "attend", "seqs": 8, "longest": 2500, "tokens": 5, "q_heads": 28, "kv_heads": 4, "page": 32, "fp32": True},
        # a whole prompt, and a chunk of a prompt far into a long one
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "longest": 2048, "tokens": 2048, "q_heads": 12, "kv_heads": 2, "page": 64, "fp32": False},
        {"name": "attend_chunk_far", "op": "attend", "seqs": 1, "longest": 32100, "tokens": 1000, "q_heads": 32, "kv_heads": 8, "page": 64, "fp32": False},
        # weights of a decode step of a batch, and of the last tokens of two long prompts
        {"name": "weights_token", "op": "weights", "seqs": 16, "longest": 4000, "tokens": 1, "q_heads": 12, "kv_heads": 2, "page": 16},
        {"name": "weights_window", "op": "weights", "seqs": 2, "longest": 32000, "tokens": 32, "q_heads": 32, "kv_heads": 8, "page": 64},
        # a conversation that ran over a small budget, and a batch of long ones
        {"name": "evict_short", "op": "evict", "seqs": 1, "longest": 1100, "q_heads": 12, "kv_heads": 2, "page": 16, "budget": 512, "sink": 4, "recent": 64},
        {"name": "evict_long", "op": "evict", "seqs": 8, "longest": 32700, "q_heads": 32, "kv_heads": 8, "page": 32, "budget": 4096, "sink": 4, "recent": 256},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "weights", "evict"])
    q, kv = rng.choice([(12, 2), (32, 8), (28, 4), (16, 4), (8, 8), (14, 2), (8, 1)])
    c = {"op": op, "q_heads": q, "kv_heads": kv, "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        tokens = _log_int(rng, 1, 4000)
        c |= {"seqs": _log_int(rng, 1, max(1, min(64, 8000 // tokens))), "tokens": tokens, "longest": tokens + _log_int(rng, 1, 4000)}
    elif op == "evict":
        longest = _log_int(rng, 100, 32000)
        budget = max(8, round(longest * rng.uniform(0.05, 0.9)))
        c |= {"seqs": _log_int(rng, 1, max(1, min(64, 250_000 // longest))), "longest": longest, "budget": budget,
              "sink": rng.randint(0, 4), "recent": rng.randint(0, budget // 2)}
    else:
        form = rng.choice(["token", "token", "few", "chunk"]) if op == "attend" else rng.choice(["token", "window"])
        longest = _log_int(rng, 30, 100_000 if form == "token" else 30_000)
        tokens = {"token": 1, "few": rng.randint(2, 8), "window": rng.randint(8, 64), "chunk": _log_int(rng, 16, 2000)}[form]
        tokens = max(1, min(tokens, longest, 30_000_000 // longest))
        most = 400_000 // longest if form in ("token", "few") else 30_000_000 // (longest * tokens)
        c |= {"seqs": _log_int(rng, 1, max(1, min(64, most))), "longest": longest, "tokens": tokens}
        if op == "attend":
            c["fp32"] = form != "chunk" and rng.random() < 0.5
    return c


def _lengths(c):
    """Cached positions of every sequence, its new ones among them, and how many are new: ragged, the first one the longest."""
    lens, new = [], []
    for i in range(c["seqs"]):
        n = max(1, round(c.get("tokens", 1) * (1 - 0.5 * math.modf(i * 0.41421356)[0])))
        lens.append(max(n, round(c["longest"] * (1 - 0.75 * math.modf(i * 0.61803399)[0]))))
        new.append(n)
    return lens, new


def work(c):
    lens, new = _lengths(c)
    q, kv, total = c["q_heads"], c["kv_heads"], sum(new)
    row = 4 * 17                                                       # bytes of a cached key or value row
    pairs = sum(n * L - n * (n - 1) // 2 for L, n in zip(lens, new))   # (query token, position it sees)
    if c["op"] == "append":                                            # q, k, v in; q and the rows out; the rows in and out as numbers
        return {"bytes": total * (2 * q * D * 2 + 2 * kv * D * 2 + 2 * kv * row * 2 + 2 * kv * D * 2), "flops": total * D * (3 * q + 12 * kv)}
    if c["op"] == "attend":
        return {"bytes": sum(lens) * kv * 2 * row + total * q * D * (2 + (4 if c["fp32"] else 2)) + total * q * 4, "flops": 4 * D * q * pairs}
    if c["op"] == "weights":
        return {"bytes": sum(lens) * kv * (row + 8) + total * q * (2 * D + 4), "flops": 2 * D * q * pairs}
    kept = sum(min(L, c["budget"]) for L in lens)
    return {"bytes": sum(lens) * kv * 4 + kept * kv * (4 * row + 4 + 4 + 4), "flops": sum(lens) * kv}


# ---- inputs --------------------------------------------------------------------------------------------------


def _quantised(x):
    """Rows [..., 128] of fp16 values -> (16 words of codes, word of scale and zero)."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).half().float()
    zero = (lo + 8 * scale).half().float()
    code = torch.where(scale > 0, torch.round((x - zero) / torch.where(scale > 0, scale, 1.0)) + 8, 8.0).clamp(0, 15).long()
    shift = torch.tensor(SHIFTS, device=x.device)
    words = (code.unflatten(-1, (16, 8)) << shift).sum(-1)
    params = (scale.half().view(torch.int16).long() & 0xFFFF) | ((zero.half().view(torch.int16).long() & 0xFFFF) << 16)
    low = lambda w: torch.where(w >= 1 << 31, w - (1 << 32), w).int()  # noqa: E731
    return low(words), low(params.squeeze(-1))


def _parts(pages, page):
    """Views of the page records: key codes, value codes [pages, heads, page, 16], key and value parameters [pages, heads, page]."""
    k, v, kp, vp = pages.split([16 * page, 16 * page, page, page], -1)
    return k.unflatten(-1, (page, 16)), v.unflatten(-1, (page, 16)), kp, vp


def prepare(c, seed):
    dev = "cuda"
    g = torch.Generator(dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    lens, new = _lengths(c)
    B, kv, q, page, total = c["seqs"], c["kv_heads"], c["q_heads"], c["page"], sum(new)
    per_seq = -(-max(lens) // page) + 1                       # one page of room, as a cache that grows has
    src = B * per_seq
    dst_per = -(-c["budget"] // page) if c["op"] == "evict" else 0
    # pages in the order in which a busy allocator hands them out; the fresh ones of an eviction behind them
    table = torch.randperm(src, generator=g, device=dev).view(B, per_seq).int()
    pages = torch.zeros(src + B * dst_per, kv, page * 34, dtype=torch.int32, device=dev)
    channel = 1 + 3 * (torch.rand(kv, D, generator=g, device=dev) < 0.04)      # keys have a few large channels
    kc, vc, kp, vp = _parts(pages[:src], page)
    step = max(1, (1 << 22) // (kv * page))
    for i in range(0, src, step):
        n = min(step, src - i)
        w, p = _quantised((randn(n, kv, page, D) * channel[:, None]).half())
        kc[i:i + n], kp[i:i + n] = w, p
        w, p = _quantised((randn(n, kv, page, D) * 0.7).half())
        vc[i:i + n], vp[i:i + n] = w, p
    lens_t, new_t = torch.tensor(lens, dtype=torch.int32, device=dev), torch.tensor(new, dtype=torch.int32, device=dev)
    start = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    start[1:] = new_t.cumsum(0)
    s = SimpleNamespace(op=c["op"], q_heads=q, scale=1 / math.sqrt(D), new_max=max(new), len_max=max(lens), new_lens=None)
    s.cache = SimpleNamespace(pages=pages, key_weight=None, num_pages=pages.shape[0], num_kv_heads=kv, page_size=page)
    s.batch = SimpleNamespace(block_table=table, seq_lens=lens_t, query_start=start if total > B else None, num_seqs=B,
                              max_pages_per_seq=per_seq, num_tokens=total)
    if c["op"] == "append":
        s.cache.key_weight = torch.ones(src, kv, page, device=dev)
        s.q, s.k, s.v = randn(total, q * D).half(), (randn(total, kv, D) * channel).half().view(total, -1), (randn(total, kv * D) * 0.7).half()
        s.q_bias, s.k_bias, s.v_bias = (randn(n * D).half() * 0.3 for n in (q, kv, kv))
        s.inv_freq = ROPE_THETA ** (-torch.arange(D // 2, device=dev, dtype=torch.float64) / (D // 2))
        s.inv_freq = s.inv_freq.float()
        s.q_out = torch.empty(total, q * D, dtype=torch.float16, device=dev)
        s.k_read, s.v_read = (torch.empty(total, kv, D, dtype=torch.float16, device=dev) for _ in range(2))
        past = torch.randint(0, 20000, (B,), generator=g, device=dev)       # positions that were evicted before
        seq = torch.repeat_interleave(torch.arange(B, device=dev), new_t)
        s.positions = (past[seq] + (lens_t - new_t)[seq] + torch.arange(total, device=dev) - start[seq]).int()
    elif c["op"] in ("attend", "weights"):
        s.q = (randn(total, q, D) * 1.2).half()
        s.lse = torch.empty(total, q, device=dev)
        if c["op"] == "attend":
            s.out = torch.empty(total, q, D, dtype=torch.float32 if c["fp32"] else torch.float16, device=dev)
            s.workspace = None                                            # made by the first call: its size is the library's to say
        else:
            s.cache.key_weight = torch.rand(src, kv, page, generator=g, device=dev)
            s.lse = _attend(s)[1]
    else:
        # what heads leave after many steps: heavy-tailed, with equal values among the little used positions
        s.cache.key_weight = torch.round(torch.exp(1.5 * randn(src + B * dst_per, kv, page) - 2) * 128) / 128
        s.cache.key_weight[src:] = 0
        s.dst_table = (src + torch.randperm(B * dst_per, generator=g, device=dev)).view(B, dst_per).int()
        s.src, s.dst_per, s.budget, s.sink, s.recent = src, dst_per, c["budget"], c["sink"], c["recent"]
        s.new_lens = torch.empty(B, dtype=torch.int32, device=dev)
        s.kept = torch.empty(B, kv, c["budget"], dtype=torch.int32, device=dev)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------


def _token_rows(b):
    """Sequence and cached position of every token of the batch."""
    if b.query_start is None:
        seq = torch.arange(b.num_seqs, device=b.seq_lens.device)
        return seq, (b.seq_lens - 1).long()
    new = (b.query_start[1:] - b.query_start[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(b.num_seqs, device=new.device), new, output_size=b.num_tokens)
    at = torch.arange(b.num_tokens, device=new.device) - b.query_start[seq]
    return seq, (b.seq_lens - new)[seq] + at


def _values(words, params):
    """Cached rows as 32-bit values."""
    shift = torch.tensor(SHIFTS, dtype=torch.int32, device=words.device)
    code = ((words.unsqueeze(-1) >> shift) & 15).flatten(-2)
    scale = (params & 0xFFFF).to(torch.int16).view(torch.float16).float().unsqueeze(-1)
    zero = ((params >> 16) & 0xFFFF).to(torch.int16).view(torch.float16).float().unsqueeze(-1)
    return (code - 8) * scale + zero


def _rotated(x, bias, cos, sin):
    x = x.float() + bias.float()
    a, b = x.unflatten(-1, (-1, D)).chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()


def _append(s):
    angle = s.positions.double()[:, None] * s.inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    s.q_out.copy_(_rotated(s.q, s.q_bias, cos, sin).flatten(1))
    k = _rotated(s.k, s.k_bias, cos, sin)
    v = (s.v.float() + s.v_bias.float()).half().unflatten(-1, (-1, D))
    page = s.cache.page_size
    seq, at = _token_rows(s.batch)
    rows = (s.batch.block_table[seq, at // page].long(), slice(None), at % page)
    kc, vc, kp, vp = _parts(s.cache.pages, page)
    kc[rows], kp[rows] = _quantised(k)
    vc[rows], vp[rows] = _quantised(v)
    s.cache.key_weight[rows] = 0
    s.k_read.copy_(_values(kc[rows], kp[rows]))
    s.v_read.copy_(_values(vc[rows], vp[rows]))
    return {"q": s.q_out, "k": s.k_read, "v": s.v_read, "key_weight": s.cache.key_weight}


def _padded(s):
    """Every sequence's rows and queries side by side, and which query sees which row."""
    b, page, dev = s.batch, s.cache.page_size, s.q.device
    at = torch.arange(s.len_max, device=dev)
    rows = (b.block_table[:, at // page].long(), slice(None), (at % page).expand(b.num_seqs, -1))
    if b.query_start is None:
        start, new = torch.arange(b.num_seqs, device=dev), torch.ones(b.num_seqs, dtype=torch.long, device=dev)
    else:
        start, new = b.query_start[:-1].long(), (b.query_start[1:] - b.query_start[:-1]).long()
    i = torch.arange(s.new_max, device=dev)
    token = (start[:, None] + i).clamp(max=b.num_tokens - 1)
    real = i < new[:, None]
    last = (b.seq_lens.long() - new)[:, None] + i
    sees = (at <= last[..., None]) & real[..., None]                     # [seqs, queries, rows]
    return rows, token, real, sees


def _scores(s, token, sees, keys):
    q = s.q.view(s.q.shape[0], -1, D)[token].float().unflatten(2, (s.cache.num_kv_heads, -1))    # [seqs, queries, kv, group, 128]
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), keys.permute(0, 2, 3, 1)) * s.scale
    x = x.unflatten(2, (-1, token.shape[1]))                              # [seqs, kv, group, queries, rows]
    return x.masked_fill_(~sees[:, None, None], -math.inf)


def _attend(s):
    rows, token, real, sees = _padded(s)
    kc, vc, kp, vp = _parts(s.cache.pages, s.cache.page_size)
    x = _scores(s, token, sees, _values(kc[rows], kp[rows]))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp_(x.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _values(vc[rows], vp[rows]).permute(0, 2, 1, 3)).unflatten(2, p.shape[2:4])
    o = o / torch.where(total > 0, total, 1.0)
    lse = (torch.log(total) + top).squeeze(-1)
    flat = lambda t: t.permute(0, 3, 1, 2, *range(4, t.dim())).flatten(2, 3)[real]  # noqa: E731  [tokens, heads, ...]
    return flat(o), flat(lse)


def _weights(s):
    rows, token, real, sees = _padded(s)
    kc, _, kp, _ = _parts(s.cache.pages, s.cache.page_size)
    x = _scores(s, token, sees, _values(kc[rows], kp[rows]))
    lse = s.lse[token].unflatten(2, (s.cache.num_kv_heads, -1)).permute(0, 2, 3, 1)[..., None]
    got = torch.exp_(x.sub_(lse)).sum((2, 3)).permute(0, 2, 1)             # [seqs, rows, kv]
    inside = sees.any(1)
    s.cache.key_weight[rows[0][inside], :, rows[2][inside]] += got[inside]
    return s.cache.key_weight


def _evict(s):
    b, page, dev = s.batch, s.cache.page_size, s.kept.device
    at = torch.arange(s.len_max, device=dev)
    src = b.block_table[:, at // page].long()
    w = s.cache.key_weight[src, :, (at % page).expand_as(src)].permute(0, 2, 1)       # [seqs, kv, rows]
    lens = b.seq_lens.long()[:, None]
    always = (at < s.sink) | (at >= lens - s.recent)
    w = torch.where(always[:, None], math.inf, w).masked_fill((at >= lens)[:, None], -math.inf)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :s.budget]
    kept_n = lens.clamp(max=s.budget)
    place = torch.arange(best.shape[-1], device=dev)
    on = (place < kept_n)[:, None].expand(-1, best.shape[1], -1)
    best = torch.where(on, best, 1 << 30).sort(-1).values
    s.kept.fill_(-1)
    s.kept[..., :best.shape[-1]] = torch.where(on, best, -1)
    s.new_lens.copy_(kept_n[:, 0])
    seq, head, j = on.nonzero(as_tuple=True)
    i = best[seq, head, j]
    old = (b.block_table[seq, i // page].long(), head, i % page)
    fresh = (s.dst_table[seq, j // page].long(), head, j % page)
    for part in (*_parts(s.cache.pages, page), s.cache.key_weight):
        part[fresh] = part[old]
    return _evicted(s)


def _evicted(s):
    # the moved rows are the same words as before, so they are given, and compared, as words
    return {"new_lens": s.new_lens, "kept": s.kept, "pages": s.cache.pages[s.src:], "key_weight": s.cache.key_weight[s.src:]}


def run(s):
    if own:
        return _own(s)
    if s.op == "attend":
        out, lse = _attend(s)
        s.out.copy_(out)
        s.lse.copy_(lse)
        return {"out": s.out, "lse": s.lse}
    return {"append": _append, "weights": _weights, "evict": _evict}[s.op](s)


def _own(s):
    import qwen_engine_b200 as lib
    if s.op == "append":
        lib.kv4_append(s.cache, s.batch, s.q, s.k, s.v, s.q_bias, s.k_bias, s.v_bias, s.positions, s.inv_freq, s.q_out, s.q_heads)
        lib.kv4_read(s.cache, s.batch, s.k_read, s.v_read)
        return {"q": s.q_out, "k": s.k_read, "v": s.v_read, "key_weight": s.cache.key_weight}
    if s.op == "attend":
        if s.workspace is None:
            n = lib.attention_kv4_workspace_bytes(s.batch.num_tokens, s.batch.num_seqs, s.q_heads, s.cache.num_kv_heads)
            s.workspace = torch.empty(n, dtype=torch.uint8, device=s.q.device)
        lib.attention_kv4(s.cache, s.batch, s.q, s.out, s.lse, s.workspace, s.q_heads, s.workspace.numel(), s.out.dtype == torch.float32, s.scale)
        return {"out": s.out, "lse": s.lse}
    if s.op == "weights":
        lib.kv4_add_key_weights(s.cache, s.batch, s.q, s.lse, s.q_heads, s.scale)
        return s.cache.key_weight
    lib.kv4_evict(s.cache, s.batch, s.dst_table, s.new_lens, s.kept, s.dst_per, s.budget, s.sink, s.recent)
    return _evicted(s)


# ---- in 64 bits, from the definitions ------------------------------------------------------------------------


def _row64(s, part, seq, head, first, n):
    """Positions first .. first + n of one sequence and head as 64-bit values; part 0 keys, 1 values."""
    page = s.cache.page_size
    at = torch.arange(first, first + n, device=s.cache.pages.device)
    record = s.cache.pages[s.batch.block_table[seq].long()[at // page], head]                # [n, page * 34]
    word = (part * page + at % page)[:, None] * 16 + torch.arange(16, device=at.device)
    codes = record.gather(1, word).long()
    both = record.gather(1, (32 * page + part * page + at % page)[:, None]).contiguous().view(torch.float16).double()
    values = torch.stack([(codes >> SHIFTS[j]) & 15 for j in range(8)], -1).flatten(1).double()
    return (values - 8) * both[:, :1] + both[:, 1:]


def exact(c, seed):
    s = prepare(c, seed)
    lens, new = _lengths(c)
    kv, group, starts = c["kv_heads"], c["q_heads"] // c["kv_heads"], [sum(new[:i]) for i in range(len(new))]
    if c["op"] == "evict":
        return None                                     # whole numbers and moved words: nothing is computed
    if c["op"] == "append":
        turn = s.positions.double()[:, None] * s.inv_freq.double()
        wave = torch.polar(torch.ones_like(turn), turn)[:, None]

        def turned(x, bias):
            x = (x.double() + bias.double()).unflatten(-1, (-1, D))
            z = torch.complex(x[..., :64], x[..., 64:]) * wave
            return torch.cat([z.real, z.imag], -1)

        def through(x):                                 # what a row reads back as
            x = x.half().double()
            lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            scale = ((hi - lo) / 15).half().double()
            zero = (lo + 8 * scale).half().double()
            return torch.clamp(torch.round((x - zero) / scale), -8, 7) * scale + zero

        weight = s.cache.key_weight.double()
        for b, (L, n) in enumerate(zip(lens, new)):
            at = torch.arange(L - n, L, device=weight.device)
            weight[s.batch.block_table[b].long()[at // c["page"]], :, at % c["page"]] = 0
        return {"q": turned(s.q, s.q_bias).flatten(1), "k": through(turned(s.k, s.k_bias)),
                "v": through((s.v.double() + s.v_bias.double()).unflatten(-1, (-1, D))), "key_weight": weight}
    q = s.q.view(-1, c["q_heads"], D).double()
    out, lse = torch.zeros_like(q), torch.zeros_like(q[..., 0])
    weight = s.cache.key_weight.double() if c["op"] == "weights" else None
    for b, (L, n) in enumerate(zip(lens, new)):
        mine = slice(starts[b], starts[b] + n)
        hidden = torch.arange(L, device=q.device) > torch.arange(L - n, L, device=q.device)[:, None]
        for h in range(kv):
            heads = slice(h * group, (h + 1) * group)
            x = torch.einsum("ngd,ld->gnl", q[mine, heads], _row64(s, 0, b, h, 0, L)) * s.scale
            x.masked_fill_(hidden, -math.inf)
            if weight is None:
                norm = torch.logsumexp(x, -1)
                lse[mine, heads] = norm.T
                out[mine, heads] = torch.einsum("gnl,ld->ngd", torch.exp(x - norm[..., None]), _row64(s, 1, b, h, 0, L))
            else:
                at = torch.arange(L, device=q.device)
                got = torch.exp(x - s.lse[mine, heads].double().T[..., None]).sum((0, 1))
                weight[s.batch.block_table[b].long()[at // c["page"]], h, at % c["page"]] += got
    return {"out": out, "lse": lse} if weight is None else weight
