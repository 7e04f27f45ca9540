"""The 4-bit key/value cache against its restatement in 64 bits (tests/kv4_reference.py): append, read, attention, attention
weights, eviction, and a run of them between the QKV and the O projection."""
import math

import numpy as np
import pytest

from tests import kv4_reference as ref
from tests import util

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
SCALE = 1 / math.sqrt(128)
BF = np.float16


@pytest.fixture(scope="module")
def ops():
    import qwen_engine_b200 as q
    q.init()
    return q


def i32(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def make(ops, seed, lens, new, kv, page, extra_pages=3, seqs_pages=None, fill=0x7FFF7FFF, bad=()):
    """A pool whose unused positions hold NaN, its twin on the device, and the batch.  bad: (sequence, page of it, number)."""
    rng = np.random.default_rng(seed)
    per = max(1, seqs_pages or -(-max(max(lens), 1) // page))
    n = len(lens) * per + extra_pages
    pool = ref.Pool(n, kv, page).fill_random(rng, 1.5, 0.7)
    table = rng.permutation(n)[:len(lens) * per].reshape(len(lens), per).astype(np.int32)
    for b, p, number in bad:
        table[b, p] = number
    used = np.zeros((n, page), bool)
    for b, L in enumerate(lens):
        for j in range(min(L, per * page)):
            if 0 <= table[b, j // page] < n:
                used[table[b, j // page], j % page] = True
    for p, s in zip(*np.nonzero(~used)):
        pool.words[p, :, 32 * page + s] = fill
        pool.words[p, :, 33 * page + s] = fill
    pool.weight[:] = rng.random(pool.weight.shape, dtype=np.float32)
    start = np.concatenate([[0], np.cumsum(new)])
    one = all(x == 1 for x in new)
    cache = ops.KV4Cache(util.to_dev(pool.words), util.to_dev(pool.weight), n, kv, page)
    batch = ops.KV4Batch.of(i32(table), i32(lens), None if one else i32(start), num_tokens=int(start[-1]))
    return rng, pool, table, cache, batch


def words_of(cache):
    return util.to_np(cache.pages, np.uint32)


# ---- append and read -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,new,kv,heads,page", [
    ([1], [1], 2, 12, 16), ([1000], [1], 2, 12, 16), ([17, 1, 33, 16], [1, 1, 1, 1], 8, 32, 16),
    ([40, 5, 0, 70], [20, 5, 0, 1], 3, 9, 32), ([129], [129], 1, 1, 64), ([5] * 70, [1] * 70, 2, 2, 16), ([300, 200], [7, 190], 8, 8, 128)])
def test_append_stores_the_formula_bit_for_bit(ops, lens, new, kv, heads, page):
    """Without rotation and bias the rows are the inputs', so codes, scales and zeros are those of the formula, whole."""
    rng, pool, table, cache, batch = make(ops, 1, lens, new, kv, page)
    T = sum(new)
    k, v = (rng.standard_normal((T, kv, 128)).astype(BF) for _ in range(2))
    k[0, 0] = 0.25                                   # a row of one value: scale 0
    v[0, 0] = np.linspace(-3e-7, 3e-7, 128)          # a scale below fp16's normal numbers
    v[-1, -1] = np.where(np.arange(128) % 2, 65504, -65504)
    want = pool.words.copy()
    for b, first, L, n in ref.spans(lens, new):
        for i in range(n):
            at = L - n + i
            for h in range(kv):
                for part, x in enumerate((k, v)):
                    w, s, z = ref.quantise(x[first + i, h])
                    pool.put(table[b, at // page], h, at % page, part, w, s, z)
                pool.weight[table[b, at // page], h, at % page] = 0
    q = rng.standard_normal((T, heads * 128)).astype(BF)
    q_out = torch.full((T, heads * 128), 7.0, dtype=torch.float16, device="cuda")
    ops.kv4_append(cache, batch, util.to_dev(q), util.to_dev(k), util.to_dev(v), None, None, None, None, None, q_out, heads)
    assert np.array_equal(words_of(cache), pool.words) and (T == 0 or not np.array_equal(want, pool.words))
    assert np.array_equal(util.to_np(cache.key_weight), pool.weight)
    assert np.array_equal(util.to_np(q_out), q)
    kr, vr = (torch.full((T + 1, kv, 128), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv4_read(cache, batch, kr, vr)
    for part, got in enumerate((kr, vr)):
        got = util.to_np(got)
        assert (got[T] == 7).all()
        for b, first, L, n in ref.spans(lens, new):
            for i in range(n):
                at = L - n + i
                for h in range(kv):
                    exact = pool.row(table[b, at // page], h, at % page, part)
                    # product exact in 32 bits, one rounding of the sum and one to fp16 (a subnormal's half step besides)
                    assert np.all(np.abs(got[first + i, h] - exact) <= np.abs(exact) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25), (part, first + i, h)


@pytest.mark.parametrize("theta,past", [(1e4, 0), (1e6, 0), (1e6, 130000)])
@pytest.mark.parametrize("strided", [False, True])
def test_append_rotates_and_adds_biases(ops, theta, past, strided):
    lens, new, kv, heads, page = [30, 9], [30, 4], 2, 6, 16
    rng, pool, table, cache, batch = make(ops, 2, lens, new, kv, page)
    T, inv = sum(new), (theta ** (-np.arange(64) / 64)).astype(np.float32)
    pos = np.concatenate([np.arange(L - n, L) for _, _, L, n in ref.spans(lens, new)]) + past
    qs, ks = heads * 128 + (64 if strided else 0), kv * 128 + (24 if strided else 0)
    q, k, v = (rng.standard_normal((T, s)).astype(BF) for s in (qs, ks, ks))
    bias = [(0.5 * rng.standard_normal(n * 128)).astype(BF) for n in (heads, kv, kv)]
    q_out = torch.full((T, qs), 7.0, dtype=torch.float16, device="cuda")
    ops.kv4_append(cache, batch, *map(util.to_dev, (q, k, v)), *map(util.to_dev, bias), i32(pos) if past else None, util.to_dev(inv), q_out, heads,
                   qs if strided else 0, ks if strided else 0)
    kr, vr = (torch.empty(T, kv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv4_read(cache, batch, kr, vr)

    def row(x, b, n):
        return (x[:, :n * 128].astype(np.float64) + b.astype(np.float64)).reshape(T, n, 128)

    want = ref.rotate(row(q, bias[0], heads), pos, inv)
    got = util.to_np(q_out)
    size = np.abs(row(q, bias[0], heads))
    size = np.concatenate([size[..., :64] + size[..., 64:]] * 2, -1)
    # one rounding to fp16; the angle's turn as fp32 (2^-25 of a turn), sine and cosine and three fp32 roundings before it
    room = size * (2 * math.pi * 2.0 ** -24 + 6 * 2.0 ** -24)
    assert np.all(np.abs(got[:, :heads * 128].reshape(T, heads, 128) - want) <= np.abs(want) * 2.0 ** -11 + room + 2.0 ** -24)
    assert (got[:, heads * 128:] == 7).all()
    for got, want in ((kr, ref.rotate(row(k, bias[1], kv), pos, inv)), (vr, row(v, bias[2], kv))):
        got = util.to_np(got).astype(np.float64)
        step = (want.max(-1, keepdims=True) - want.min(-1, keepdims=True)) / 15
        big = np.abs(want).max(-1, keepdims=True)
        # half a step, the scale's rounding 7.5 steps from the zero, and the zero's, the row's and the output's roundings
        assert np.all(np.abs(got - want) <= step * (0.5 + 8 * 2.0 ** -11) + 3 * big * 2.0 ** -11 + 1e-6)


def test_append_leaves_alone_what_it_may_not_touch(ops):
    """Rows behind the last sequence, positions past the table, page numbers outside the pool, a row with an infinity."""
    lens, new, kv, heads, page = [20, 40, 34], [4, 8, 2], 2, 2, 16
    rng, pool, table, cache, batch = make(ops, 3, lens, new, kv, page, seqs_pages=2, bad=[(2, 1, 10 ** 6), (0, 0, -5)])
    T = sum(new) + 3
    batch.num_tokens = T
    k, v = (rng.standard_normal((T, kv, 128)).astype(BF) for _ in range(2))
    k[1, 1, 5], v[2, 0, 127] = np.inf, np.nan
    q = rng.standard_normal((T, heads * 128)).astype(BF)
    q_out = torch.full((T, heads * 128), 7.0, dtype=torch.float16, device="cuda")
    for b, first, L, n in ref.spans(lens, new):
        for i in range(n):
            at = L - n + i
            if at < 2 * page and 0 <= table[b, at // page] < pool.num_pages:
                for h in range(kv):
                    for part, x in enumerate((k, v)):
                        w, s, z = ref.quantise(x[first + i, h])
                        pool.put(table[b, at // page], h, at % page, part, w, s, z)
                    pool.weight[table[b, at // page], h, at % page] = 0
    ops.kv4_append(cache, batch, util.to_dev(q), util.to_dev(k), util.to_dev(v), None, None, None, None, None, q_out, heads)
    got = words_of(cache).copy()
    ps = page
    for a in (got, pool.words):     # NaNs of any payload are the same
        p = a[..., 32 * ps:].view(np.uint16)
        p[(p & 0x7FFF) > 0x7C00] = 0x7E00
    assert np.array_equal(got, pool.words)
    assert np.array_equal(util.to_np(cache.key_weight), pool.weight)
    assert (util.to_np(q_out)[sum(new):] == 7).all() and np.array_equal(util.to_np(q_out)[:sum(new)], q[:sum(new)])
    kr = torch.full((T, kv, 128), 7.0, dtype=torch.float16, device="cuda")
    ops.kv4_read(cache, batch, kr, None)
    kr = util.to_np(kr)
    assert np.isnan(kr[1, 1]).all() and np.isfinite(kr[1, 0]).all()
    assert (kr[sum(new):] == 7).all()
    assert (kr[4:12][[i for i in range(8) if 40 - 8 + i >= 32]] == 0).all() and (kr[12:14] == 0).all()


def test_append_of_rows_with_few_steps_or_subnormal_scales(ops):
    """Rows of one to forty steps of fp16 far from zero, where zero's rounding is up to 7.5 scales, and rows whose scale is subnormal and up to
    half a step off: quotients go to 15 and beyond, and the codes are the formula's all the same."""
    kv, page, T = 4, 16, 64
    rng, pool, table, cache, batch = make(ops, 23, [T], [T], kv, page)
    x = np.empty((2, T, kv, 128), BF)
    for part in range(2):
        for t in range(T):
            for h in range(kv):
                steps = int(rng.integers(1, 41))
                if (t + h) % 2:
                    base = int(rng.integers(0x0400, 0x7800))                 # bits of a normal number and of those above it
                    x[part, t, h] = (base + rng.integers(0, steps + 1, 128)).astype(np.uint16).view(BF) * BF(rng.choice([-1, 1]))
                else:                                                        # multiples of 2^-24
                    x[part, t, h] = (rng.integers(-4 * steps, 4 * steps + 1, 128) * 2.0 ** -24 + rng.choice([0, 2.0 ** -14])).astype(BF)
    x[0, 0, 0] = 1.0 + 2.0 ** -10 * (np.arange(128) % 2)
    most = 0.0
    for t in range(T):
        for h in range(kv):
            for part in range(2):
                w, s, z = ref.quantise(x[part, t, h])
                pool.put(table[0, t // page], h, t % page, part, w, s, z)
                if s > 0:
                    most = max(most, np.abs((x[part, t, h].astype(np.float64) - float(z)) / float(s)).max())
    assert 14 < most < 23
    ops.kv4_append(cache, batch, None, util.to_dev(x[0]), util.to_dev(x[1]), None, None, None, None, None, None)
    assert np.array_equal(words_of(cache), pool.words)


@pytest.mark.parametrize("kv", [5, 8])
def test_append_of_keys_and_values_alone(ops, kv):
    """No queries, and numbers of heads that are no divisors of the default number of query heads."""
    lens, new, page = [20, 33], [20, 2], 16
    rng, pool, table, cache, batch = make(ops, 22, lens, new, kv, page)
    k, v = (rng.standard_normal((22, kv, 128)).astype(BF) for _ in range(2))
    for b, first, L, n in ref.spans(lens, new):
        for i in range(n):
            at = L - n + i
            for h in range(kv):
                for part, x in enumerate((k, v)):
                    pool.put(table[b, at // page], h, at % page, part, *ref.quantise(x[first + i, h]))
    ops.kv4_append(cache, batch, None, util.to_dev(k), util.to_dev(v), None, None, None, None, None, None)
    assert np.array_equal(words_of(cache), pool.words)


# ---- attention -----------------------------------------------------------------------------------------------------------


def attend(ops, cache, batch, q, heads, f32, scale=SCALE, q_stride=0, lse=True):
    T = batch.num_tokens
    out = torch.full((T + 1, heads, 128), 7.0, dtype=torch.float32 if f32 else torch.float16, device="cuda")
    l = torch.full((T + 1, heads), 7.0, device="cuda") if lse else None
    n = ops.attention_kv4_workspace_bytes(T, batch.num_seqs, heads, cache.num_kv_heads)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") if n else None       # NaNs: nothing in it may be read unwritten
    ops.attention_kv4(cache, batch, q, out, l, ws, heads, n, f32, scale, q_stride)
    return util.to_np(out), util.to_np(l) if lse else None


SHAPES = [
    ([1], [1], 2, 12, 16), ([16], [1], 2, 12, 16), ([17], [1], 1, 1, 16), ([1021], [1], 2, 12, 16), ([2500], [1], 2, 14, 64),
    ([5, 0, 33, 64, 65, 127], [1] * 6, 2, 2, 32), ([100] * 40, [1] * 40, 8, 32, 16), ([200, 77], [1, 1], 1, 20, 16),
    ([30, 12, 9, 0], [5, 1, 0, 0], 4, 28, 16), ([300], [3], 1, 16, 128), ([65, 64, 63], [65, 1, 30], 2, 4, 16), ([7], [20], 2, 4, 16),
    ([190, 250], [130, 250], 1, 3, 64),
    ([260], [40], 2, 16, 16), ([513, 3, 129, 0], [200, 3, 1, 0], 2, 4, 32), ([700], [33], 1, 8, 128), ([128, 127], [128, 127], 1, 2, 16),
]


def few_rows(batch, heads, cache, f32):
    """Whether a call takes the form that never rounds a value: 32-bit results, or under 64 query rows a sequence."""
    return f32 or heads // cache.num_kv_heads * batch.num_tokens < 64 * batch.num_seqs


def check_attention(got, lse, want, T, f32):
    out, wl, eout, el = want
    # the bounds are the worst case; as a whole the result is nearer: roundings to fp16 are at most 2^-11 of a value and 2^-12.3 on
    # average, those of values, weights and the result together 2^-11.5
    assert np.linalg.norm(got[:T] - out) <= (2.0 ** -18 if f32 else 2.0 ** -10.5) * np.linalg.norm(out)
    room = eout if f32 else eout + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    off = np.abs(got[:T] - out)
    assert np.all(off <= room), (off.max(), (off / np.maximum(room, 1e-30)).max())
    assert (got[T] == 7).all()
    if lse is not None:
        empty = np.isneginf(wl)
        assert np.array_equal(np.isneginf(lse[:T]), empty) and (lse[T] == 7).all()
        assert np.all(np.abs(lse[:T][~empty] - wl[~empty]) <= el[~empty])


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("lens,new,kv,heads,page", SHAPES)
def test_attention(ops, lens, new, kv, heads, page, f32):
    rng, pool, table, cache, batch = make(ops, 4, lens, new, kv, page)
    q = (1.2 * rng.standard_normal((batch.num_tokens, heads, 128))).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q, SCALE, not few_rows(batch, heads, cache, f32)), batch.num_tokens, f32)


@pytest.mark.parametrize("new,f32", [([1, 1, 1], True), ([4, 2, 40], True), ([50, 30, 40], False)])
def test_attention_does_not_see_what_it_may_not(ops, new, f32):
    """Page numbers outside the pool, positions past the table; tokens behind the last sequence stay; strided q; no lse."""
    lens, kv, heads, page = [60, 50, 70], 2, 6, 16
    rng, pool, table, cache, batch = make(ops, 5, lens, new, kv, page, seqs_pages=4, bad=[(0, 1, -1), (1, 3, 1 << 30), (2, 0, 10 ** 5)])
    T = sum(new)
    q = np.full((T, heads * 128 + 8), np.nan, BF)
    q[:, :heads * 128] = (1.2 * rng.standard_normal((T, heads * 128))).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32, lse=False, q_stride=heads * 128 + 8)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q[:, :heads * 128].reshape(T, heads, 128), SCALE, not f32), T, f32)


@pytest.mark.parametrize("heads,f32", [(4, True), (40, True), (40, False)])
def test_a_poisoned_row_reaches_the_tokens_that_see_it_only(ops, heads, f32):
    lens, new, kv, page = [50], [20], 1, 16
    rng, pool, table, cache, batch = make(ops, 6, lens, new, kv, page)
    q = rng.standard_normal((20, heads, 128)).astype(BF)
    for part in range(2):
        clean = cache.pages.clone()
        slot = 40 % page
        cache.pages[int(table[0, 40 // page]), 0, (32 + part) * page + slot] = 0x7E007E00
        got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
        want = ref.attention(pool, table, lens, new, q, SCALE, not f32)
        # token i is position 30 + i: those from 10 on see position 40
        assert np.isnan(got[10:20]).all()
        assert np.all(np.abs(got[:10] - want[0][:10]) <= want[2][:10] + (0 if f32 else np.abs(want[0][:10]) * 2.0 ** -11 + 2.0 ** -25))
        cache.pages.copy_(clean)


@pytest.mark.parametrize("tokens,heads,f32", [(2, 2, False), (70, 2, False), (300, 4, False), (2, 2, True)])
def test_attention_over_the_largest_values_is_finite(ops, tokens, heads, f32):
    """Rows from -65504 to 65504 come back as -65504 to 65536 (scale 8736, zero 4384: -8 * 8736 + 4384, 7 * 8736 + 4384), which is no fp16
    number: fp16 results end at 65504, as rows that are read do.

    Every position has the same values, so the average is theirs: for 32 bits but for sums; for fp16 results but for weights and result, 2^-11
    each; in the chunk form the value besides, and its scale and zero, which are 65504 / 65536 as large (2^-11) and cut to fp16 (2^-10)."""
    kv, page, n = 1, 16, 300
    rng, pool, table, cache, batch = make(ops, 24, [n], [tokens], kv, page)
    x = np.where(np.arange(128) % 2, 65504, -65504).astype(BF)
    for j in range(n):
        pool.put(table[0, j // page], 0, j % page, 1, *ref.quantise(x))
    assert np.abs(pool.rows(table[0], 0, n, 1)[0]).max() == 65536
    cache.pages.copy_(util.to_dev(pool.words))
    q = (3 * rng.standard_normal((tokens, heads, 128))).astype(BF)
    got, _ = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    got = got[:tokens].astype(np.float64)
    assert np.isfinite(got).all() and np.all(np.sign(got) == np.sign(x.astype(np.float64)))
    v = pool.row(table[0, 0], 0, 0, 1)
    room = 2.0 ** -18 if f32 else 2.0 ** -10 if few_rows(batch, heads, cache, f32) else 3 * 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -10
    assert np.all(np.abs(got - (v if f32 else np.clip(v, -65504, 65504))) <= 65504 * room)


@pytest.mark.parametrize("tokens,f32", [(2, True), (9, True), (2, False), (100, False)])
@pytest.mark.parametrize("high", [10.2, 20.4, 22.7, 23.3, 23.8, 24.6, 25.3, 26.5, 27.4, 28.3, 28.9, 30.6, 33.1])
def test_attention_with_scores_that_are_far_above_what_32_bits_count_in(ops, high, tokens, f32):
    """Scores of about 2^high in the exponent's base: from 2^24 on neighbouring 32-bit numbers are more than 1 apart, so the reference of the exponents
    cannot be chosen freely.  A few positions share the largest score bit for bit (their key rows are the same), with values of every
    size, and all others are far below: the result is the average of those.

    It is off by the weights' and values' roundings alone, relative to what makes it up: two fp16 parts 2^-21, with the sums 2^-18; one 2^-11, and
    the value's 2^-11 in the chunk form.  lse: a score's sum, scaling and logarithm, at most 2^-21 of it."""
    n, kv, heads, page = 300, 1, 2, 16
    rng, pool, table, cache, batch = make(ops, 25, [n], [tokens], kv, page)
    c, first = 60000.0, {0: [3, 17, 66, 140, 190], 1: [1, 40, 64, 65, 199]}
    scale = 2.0 ** high * math.log(2) / (c * 50000.0)
    top = rng.uniform(-0.9, 0.9, 128) * c
    size = [1.0, 1e-3, 0.0, 30.0, 3e3]
    for j in range(n):
        k = rng.uniform(-0.8, 0.8, 128) * c
        v = rng.standard_normal(128)
        for h in range(2):
            if j in first[h]:
                k = np.concatenate([[c * (1, -1)[h]], top[1:]])
                v = v * size[first[h].index(j)] + 0.125
        for part, x in enumerate((k, v)):
            pool.put(table[0, j // page], 0, j % page, part, *ref.quantise(x.astype(BF)))
    cache.pages.copy_(util.to_dev(pool.words))
    q = np.zeros((tokens, heads, 128), BF)
    q[:, 0, 0], q[:, 1, 0] = 50000, -50000
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32, scale)
    k, v = (pool.rows(table[0], 0, n, part)[0] for part in range(2))
    p = np.concatenate([pool.words[x, 0, 33 * page:34 * page] for x in table[0]])[:n]
    vs, vz = ((p & 0xFFFF).astype(np.uint16).view(BF).astype(np.float64), (p >> 16).astype(np.uint16).view(BF).astype(np.float64))
    few = few_rows(batch, heads, cache, f32)
    for h in range(2):
        D = first[h]
        want, made_of = v[D].mean(0), (7.5 * vs + np.abs(vz - vs / 2))[D].mean()
        room = made_of * (2.0 ** -18 if f32 else 2.0 ** -11 if few else 2.0 ** -10) + (0 if f32 else np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
        for i in range(tokens):
            assert np.all(np.abs(got[i, h] - want) <= room), (i, h, np.abs(got[i, h] - want).max() / np.max(room))
            wl = k[D[0], 0] * float(q[i, h, 0]) * scale + math.log(len(D))
            assert abs(lse[i, h] - wl) <= 2.0 ** -21 * abs(wl), (i, h, lse[i, h] / wl - 1)


@pytest.mark.parametrize("sign", [0, 0x80008000])
@pytest.mark.parametrize("heads,f32", [(4, True), (4, False), (40, False)])
def test_a_poisoned_key_makes_lse_of_the_tokens_that_see_it_nan(ops, heads, f32, sign):
    lens, new, kv, page = [300], [20], 1, 16
    rng, pool, table, cache, batch = make(ops, 26, lens, new, kv, page)
    q = rng.standard_normal((20, heads, 128)).astype(BF)
    cache.pages[int(table[0, 290 // page]), 0, 32 * page + 290 % page] = int(np.uint32(0x7E007E00 | sign).view(np.int32))
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    want = ref.attention(pool, table, lens, new, q, SCALE, not few_rows(batch, heads, cache, f32))
    # token i is position 280 + i
    assert np.isnan(lse[10:20]).all() and np.isnan(got[10:20]).all()
    assert np.all(np.abs(lse[:10] - want[1][:10]) <= want[3][:10]) and np.isfinite(got[:10]).all()


@pytest.mark.parametrize("heads,f32", [(4, True), (4, False), (40, False)])
def test_a_poisoned_value_leaves_lse_and_weights_alone(ops, heads, f32):
    """The logarithm of the sum and the attention weights come from queries and keys: a value row of NaNs reaches the outputs only."""
    lens, new, kv, page = [300], [20], 1, 16
    rng, pool, table, cache, batch = make(ops, 19, lens, new, kv, page)
    q = rng.standard_normal((20, heads, 128)).astype(BF)
    for at in (5, 285):
        cache.pages[int(table[0, at // page]), 0, 33 * page + at % page] = 0x7E007E00
    want = ref.attention(pool, table, lens, new, q, SCALE, not few_rows(batch, heads, cache, f32))
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    assert np.isnan(got[:20]).all()
    assert np.all(np.abs(lse[:20] - want[1]) <= want[3])
    add, rel = ref.key_weights(pool, table, lens, new, q, lse[:20].astype(np.float64), SCALE)
    ops.kv4_add_key_weights(cache, batch, util.to_dev(q), util.to_dev(lse[:20]), heads, SCALE)
    total = pool.weight + add
    assert np.all(np.abs(util.to_np(cache.key_weight) - total) <= add * rel + total * 2.0 ** -22)


@pytest.mark.parametrize("factor", [1e-3, 1.0, 3e3])
@pytest.mark.parametrize("tokens,f32", [(1, True), (1, False), (40, False)])
def test_attention_of_values_of_any_size(ops, factor, tokens, f32):
    """Value scales from 2^-14 to above 2^10, and a few rows that are larger by a thousand: the weights' power of two follows."""
    lens, new, kv, heads, page = [700], [tokens], 1, 4, 16
    rng, pool, table, cache, batch = make(ops, 7, lens, new, kv, page)
    for page_no in table[0]:
        for s in range(page):
            x = (rng.standard_normal(128) * factor * (1.0 if rng.random() < 0.95 else 5.0 if factor > 1 else 1000.0)).astype(BF)
            pool.put(page_no, 0, s, 1, *ref.quantise(x))
    cache.pages.copy_(util.to_dev(pool.words))
    q = rng.standard_normal((tokens, heads, 128)).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q, SCALE, not few_rows(batch, heads, cache, f32)), tokens, f32)


@pytest.mark.parametrize("tokens,f32", [(2, True), (2, False), (30, False)])
def test_attention_with_steep_scores(ops, tokens, f32):
    """Scores in the hundreds, rising along the sequence, so that the running maximum keeps moving."""
    lens, new, kv, heads, page = [600], [tokens], 1, 4, 32
    rng, pool, table, cache, batch = make(ops, 8, lens, new, kv, page)
    direction = rng.standard_normal(128)
    for j in range(600):
        x = (direction * (j / 60) + 0.1 * rng.standard_normal(128)).astype(BF)
        pool.put(table[0, j // page], 0, j % page, 0, *ref.quantise(x))
    cache.pages.copy_(util.to_dev(pool.words))
    q = (direction * np.array([1, -1, 3, -3])[:, None] + np.zeros((tokens, 4, 128))).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    want = ref.attention(pool, table, lens, new, q, SCALE, not few_rows(batch, heads, cache, f32))
    check_attention(got, lse, want, tokens, f32)


@pytest.mark.parametrize("tokens,f32", [(100, False), (3, False), (3, True)])
def test_attention_of_queries_as_large_as_fp16_goes(ops, tokens, f32):
    """Rows whose sum passes 524 032 (eight times fp16's end), up to 128 times the end, beside ordinary ones; a scale that keeps scores small."""
    lens, new, kv, heads, page, scale = [300], [tokens], 1, 4, 16, 1e-5
    rng, pool, table, cache, batch = make(ops, 16, lens, new, kv, page)
    q = rng.standard_normal((tokens, heads, 128))
    q[:, 1] = 4500 + 100 * q[:, 1]
    q[:, 2] = -30000 + 9000 * q[:, 2]
    q[0, 3], q[1, 3] = 65504, -65504
    q[2, 3, :64] = 60000                                  # and tiny elements beside large ones
    q = np.clip(q, -65504, 65504).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32, scale)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q, scale, not few_rows(batch, heads, cache, f32)), tokens, f32)


@pytest.mark.parametrize("tokens,f32", [(100, False), (3, False), (3, True)])
def test_attention_over_keys_that_span_the_whole_of_fp16(ops, tokens, f32):
    """Key scales around 8188, eight times which is fp16's end, up to 8736; a softmax scale that keeps scores small."""
    lens, new, kv, heads, page, scale = [300], [tokens], 1, 4, 16, 1e-6
    rng, pool, table, cache, batch = make(ops, 17, lens, new, kv, page)
    for j in range(300):
        x = rng.uniform(-1, 1, 128) * [65504, 61440, 3.0][j % 3]
        x[:2] = np.abs(x).max() * np.array([1, -1])
        x[2] = rng.uniform(-65504, 65504) if j % 7 == 0 else x[2]
        pool.put(table[0, j // page], 0, j % page, 0, *ref.quantise(x.astype(BF)))
    cache.pages.copy_(util.to_dev(pool.words))
    q = rng.standard_normal((tokens, heads, 128)).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32, scale)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q, scale, not few_rows(batch, heads, cache, f32)), tokens, f32)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("tokens,heads", [(2, 4), (3, 4)])
@pytest.mark.parametrize("gap", [2, 16, 20, 24, 40])
@pytest.mark.parametrize("first", ["zero", "tiny", "large", "behind"])
def test_attention_keeps_what_counts_in_the_result(ops, first, gap, tokens, heads, f32):
    """A first position ahead by `gap` in the score (for one head as far behind) with values of none, of 1e-4 or of 1e4 of the size of the
    others', or a few early ones as far behind with values 1e6 as large; and a last one, seen by the last token alone, with such values:
    results are off relative to what the weights and values that make them up come to, not to the largest weight or value of the cache.

    Queries have one element, so a score is one product: exact but for the scaling, the zero's part and their sum, 2^-24 each of their
    sizes, and the exponent's argument, 2^-24 of it (the scores' range and up to 55 for the value scales'): d.  A weight is off by 2 d, so is their sum; the exponential adds 2^-22, two
    fp16 parts 2^-21 (one: 2^-11), 32-bit sums of a row's L terms in groups of 16, truncated, L 2^-27, and the parts' joins 8 roundings."""
    lens, new, kv, page = [700], [tokens], 1, 16
    rng, pool, table, cache, batch = make(ops, 18, lens, new, kv, page)
    size = {"zero": 0.0, "tiny": 1e-4, "large": 1e4, "behind": 0.01}[first]
    others, behind = 0.01 if first == "behind" else 1.0, (3, 19, 35, 51) if first == "behind" else ()
    for j in range(700):
        k = 0.2 * rng.standard_normal(128) * (10 if behind else 1)       # there a few positions get most of the rest
        k[0] = -8.0 if j in behind else 8.0 if j == 0 and not behind else k[0]
        v = rng.standard_normal(128) * (size if j == 0 else 1e4 if j == 699 or j in behind else others) + (others / 2 if j % 50 == 1 else 0.0)
        if j % 97 == 5:
            v[:] = 0.25                                  # a scale of zero
        for part, x in enumerate((k, v)):
            pool.put(table[0, j // page], 0, j % page, part, *ref.quantise(x.astype(BF)))
    cache.pages.copy_(util.to_dev(pool.words))
    q = np.zeros((tokens, heads, 128), BF)
    q[:, :, 0] = gap / 8 / SCALE * np.array([1, 0.9, -1, 0.8])
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    k, v = (pool.rows(table[0], 0, 700, part)[0] for part in range(2))
    params = [np.concatenate([pool.words[p, 0, (32 + part) * page:(33 + part) * page] for p in table[0]])[:700] for part in range(2)]
    scale, zero = zip(*[((p & 0xFFFF).astype(np.uint16).view(BF).astype(np.float64), (p >> 16).astype(np.uint16).view(BF).astype(np.float64)) for p in params])
    for i in range(tokens):
        n = 700 - tokens + i + 1
        for h in range(heads):
            x = float(q[i, h, 0])
            s = k[:n, 0] * x * SCALE
            p = np.exp(s - s.max())
            d = 3 * 2.0 ** -24 * (8 * scale[0][:n] + np.abs(zero[0][:n])).max() * abs(x) * SCALE + ((s.max() - s.min()) * 1.45 + 55 + 2 * np.abs(s).max()) * 2.0 ** -24
            made_of = p @ (7.5 * scale[1][:n] + np.abs(zero[1][:n] - scale[1][:n] / 2)) / p.sum()
            want = p @ v[:n] / p.sum()
            room = made_of * (4 * d + 2.0 ** -22 + (2.0 ** -21 if f32 else 2.0 ** -11) + n * 2.0 ** -27 + 8 * 2.0 ** -24)
            room = room + (0 if f32 else np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
            assert np.all(np.abs(got[i, h] - want) <= room), (i, h, np.abs(got[i, h] - want).max() / np.max(room))
            wl = s.max() + np.log(p.sum())
            assert abs(lse[i, h] - wl) <= 2 * d + 2.0 ** -21 + 2.0 ** -22 * abs(wl), (i, h, lse[i, h] - wl)


# ---- weights and eviction ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,new,kv,heads,page", SHAPES)
def test_key_weights(ops, lens, new, kv, heads, page):
    rng, pool, table, cache, batch = make(ops, 9, lens, new, kv, page)
    q = (1.2 * rng.standard_normal((batch.num_tokens, heads, 128))).astype(BF)
    lse = ref.attention(pool, table, lens, new, q, SCALE)[1].astype(np.float32)
    add, rel = ref.key_weights(pool, table, lens, new, q, lse.astype(np.float64), SCALE)
    for turn in range(2):
        ops.kv4_add_key_weights(cache, batch, util.to_dev(q), util.to_dev(lse), heads, SCALE)
        want = pool.weight + (turn + 1) * add
        got = util.to_np(cache.key_weight)
        assert np.all(np.abs(got - want) <= add * 2 * rel + np.abs(want) * 2.0 ** -22), turn
        assert np.array_equal(got[add == 0], pool.weight[add == 0])


@pytest.mark.parametrize("lens,kv,page,budget,sink,recent", [
    ([100], 2, 16, 33, 4, 8), ([5, 0, 64, 65, 200], 1, 16, 64, 0, 0), ([1100], 2, 16, 512, 4, 64), ([3000, 2999], 3, 64, 1, 0, 1),
    ([4000], 1, 128, 3999, 2, 5), ([50], 2, 16, 20, 10, 10), ([9000], 1, 32, 700, 4, 256), ([40000], 2, 64, 5000, 4, 256)])
@pytest.mark.parametrize("kind", ["random", "equal", "odd"])
def test_eviction(ops, lens, kv, page, budget, sink, recent, kind):
    bad = [(0, 1, -3)] if kind == "odd" and max(lens) > page else []
    rng, pool, table, cache, batch = make(ops, 10, lens, [1] * len(lens), kv, page, fill=0x3C003C00, bad=bad)
    if kind == "equal":
        pool.weight[:] = np.round(pool.weight * 3) / 3
    elif kind == "odd":
        pool.weight[:] = np.exp(8 * rng.standard_normal(pool.weight.shape)) * rng.choice([1, -1, 0, -0.0], pool.weight.shape)
        pool.weight[rng.random(pool.weight.shape) < 0.1] = np.nan
        pool.weight[rng.random(pool.weight.shape) < 0.05] = np.inf
    cache.key_weight.copy_(util.to_dev(pool.weight))
    B, per = len(lens), -(-budget // page)
    n = pool.num_pages
    cache = ops.KV4Cache(torch.cat([cache.pages, torch.full_like(cache.pages[:1], 9).expand(B * per, -1, -1)]),
                         torch.cat([cache.key_weight, torch.full((B * per, kv, page), 9.0, device="cuda")]), n + B * per, kv, page)
    dst = n + rng.permutation(B * per).reshape(B, per)
    new_lens, kept = i32(np.full(B, 77)), i32(np.full((B, kv, budget), 77))
    ops.kv4_evict(cache, batch, i32(dst), new_lens, kept, per, budget, sink, recent)
    words, weight, kept = words_of(cache), util.to_np(cache.key_weight), util.to_np(kept)
    assert np.array_equal(words[:n], pool.words) and np.array_equal(weight[:n], pool.weight, equal_nan=True)
    assert util.to_np(new_lens).tolist() == [min(L, budget) for L in lens]
    for b, L in enumerate(lens):
        for h in range(kv):
            want = ref.evict(pool.weight, table[b], L, h, page, n, budget, sink, recent)
            assert kept[b, h].tolist() == want + [-1] * (budget - len(want)), (b, h)
            for j in range(per * page):
                rec, slot = words[dst[b, j // page], h], j % page
                old = want[j] if j < len(want) else None
                page_no = table[b, old // page] if old is not None else -1
                for part in range(2):
                    mine = np.append(rec[(part * page + slot) * 16:][:16], rec[(32 + part) * page + slot])
                    if 0 <= page_no < n:
                        src, s = pool.words[page_no, h], old % page
                        assert np.array_equal(mine, np.append(src[(part * page + s) * 16:][:16], src[(32 + part) * page + s]))
                    else:
                        assert (mine == 9).all()
                if 0 <= page_no < n:
                    assert np.array_equal(weight[dst[b, j // page], h, slot], pool.weight[page_no, h, old % page], equal_nan=True)
                else:
                    assert weight[dst[b, j // page], h, slot] == 9


def check_eviction(ops, lens, kv, page, budget, sink, recent, weight_of, stale=0x7FFFFFFF):
    """An eviction of sequences on pages of the pool, whole records compared.  `stale`: what the list of kept positions holds before."""
    rng = np.random.default_rng(30)
    B, per, dst_per = len(lens), -(-max(lens) // page), -(-budget // page)
    n = B * (per + dst_per)
    table = rng.permutation(n).reshape(B, per + dst_per).astype(np.int32)
    table, dst = table[:, :per].copy(), table[:, per:].copy()
    words = rng.integers(0, 1 << 32, (n, kv, 34 * page), dtype=np.uint32)
    weight = weight_of(rng, (n, kv, page)).astype(np.float32)
    cache = ops.KV4Cache(util.to_dev(words), util.to_dev(weight), n, kv, page)
    new_lens, kept = i32(np.full(B, 77)), i32(np.full((B, kv, budget), stale))
    ops.kv4_evict(cache, ops.KV4Batch.of(i32(table), i32(lens)), i32(dst), new_lens, kept, dst_per, budget, sink, recent)
    got_words, got_weight, kept = words_of(cache), util.to_np(cache.key_weight), util.to_np(kept)
    assert util.to_np(new_lens).tolist() == [min(L, budget) for L in lens]
    for b, L in enumerate(lens):
        for h in range(kv):
            want = np.array(ref.evict(weight, table[b], L, h, page, n, budget, sink, recent), dtype=np.int64)
            assert np.array_equal(kept[b, h], np.append(want, np.full(budget - len(want), -1))), (b, h)
            new = np.arange(len(want))
            from_, to = (table[b, want // page], h, want % page), (dst[b, new // page], h, new % page)
            for part in range(2):
                codes = slice(part * 16 * page, (part + 1) * 16 * page)
                view = lambda w: w[..., codes].reshape(n, kv, page, 16)  # noqa: E731
                assert np.array_equal(view(got_words)[to], view(words)[from_])
                params = slice((32 + part) * page, (33 + part) * page)
                assert np.array_equal(got_words[..., params][to], words[..., params][from_])
            assert np.array_equal(got_weight[to], weight[from_], equal_nan=True)


@pytest.mark.parametrize("budget", [65, 700, 1500, 2200, 2990])
@pytest.mark.parametrize("kind", ["low", "zeros", "high", "wide"])
def test_eviction_of_weights_at_the_ends_of_the_searchs_first_range(ops, budget, kind):
    """Weights densely around 2^-32 (what a peaked head leaves to most positions) and 2^32, where the first histogram's bins end."""
    def weights(rng, shape):
        if kind == "zeros":
            return rng.uniform(1.0, 1.3, shape) * 2.0 ** -32 * rng.choice([0, 1, 1], shape)
        if kind == "wide":
            return np.exp(rng.uniform(-40, 0, shape))
        return 2.0 ** rng.uniform(-1, 1, shape) * 2.0 ** (32 if kind == "high" else -32)
    check_eviction(ops, [3000, 2500], 2, 16, budget, 4, 60, weights)


@pytest.mark.parametrize("budget,sink,recent", [(300, 4, 64), (135000, 0, 1)])
def test_eviction_of_more_positions_than_shared_memory_holds(ops, budget, sink, recent):
    """From 131 072 positions on a CTA of the cluster reads its weights again in every pass."""
    check_eviction(ops, [140001, 131500, 100], 1, 128, budget, sink, recent, lambda rng, shape: np.round(np.exp(9 * rng.standard_normal(shape)), 3))


# ---- as they are used ----------------------------------------------------------------------------------------------------


def test_decode_steps_between_qkv_and_o(ops):
    """QKV projection -> append -> attention (fp32 heads) -> O projection from the heads, captured once and replayed while the
    sequence grows; then weights, eviction, and attention over what is left."""
    from qwen_engine_b200 import synth
    H, heads, kv, page, steps = 1536, 12, 2, 16, 40
    dev = lambda a: util.to_dev(a)  # noqa: E731
    W = {n: (dev(synth.packed_weights(1, n, r, H)), dev(synth.scales(1, n, r, H))) for n, r in (("q", H), ("k", 256), ("v", 256), ("o", H))}
    h = dev(synth.activations(1, "h", H))
    gamma = torch.full((H,), 0.05, dtype=torch.float16, device="cuda")
    bufs = {n: torch.empty(r, dtype=torch.float16, device="cuda") for n, r in (("q", H), ("k", 256), ("v", 256), ("o", H))}
    view = ops.QKVProjectionView(*W["q"], bufs["q"], *W["k"], bufs["k"], *W["v"], bufs["v"])
    per = 4
    cache = ops.KV4Cache.allocate(2 * per, page, kv, key_weight=True)
    table, lens = i32(np.arange(per)[None, ::-1].copy()), i32([0])
    batch = ops.KV4Batch.of(table, lens)
    inv = torch.tensor(1e6 ** (-np.arange(64) / 64), dtype=torch.float32, device="cuda")
    acc, lse = torch.empty(1, heads, 128, device="cuda"), torch.empty(1, heads, device="cuda")
    n = ops.attention_kv4_workspace_bytes(1, 1, heads, kv)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out = torch.empty(H, dtype=torch.float16, device="cuda")

    def step():
        lens.add_(1)
        ops.launch_gemv_qkv_rmsnorm_w4a16(view, h, gamma, in_features=H, num_q_heads=heads, num_kv_heads=kv)
        ops.kv4_append(cache, batch, bufs["q"], bufs["k"], bufs["v"], None, None, None, None, inv, bufs["q"], heads)
        ops.attention_kv4(cache, batch, bufs["q"], acc, lse, ws, heads, n, True, SCALE)
        ops.gemv_attn_heads_f32_w4a16(*W["o"], acc, h, out, H, H)
        ops.kv4_add_key_weights(cache, batch, bufs["q"], lse, heads, SCALE)
        h.copy_(out)

    h0 = h.clone()
    step()                                       # eager, then captured
    stream = torch.cuda.Stream()
    lens.zero_(), h.copy_(h0), cache.pages.zero_(), cache.key_weight.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    seen = []
    for _ in range(steps):
        before = h.clone()
        graph.replay()
        torch.cuda.synchronize()
        seen.append((before, bufs["q"].clone(), acc.clone(), out.clone(), lse.clone()))
    assert lens.item() == steps
    pool = ref.Pool(2 * per, kv, page)
    pool.words[:] = words_of(cache)
    total = np.zeros_like(pool.weight, dtype=np.float64)
    for i in (0, 1, 15, 16, steps - 1):
        before, q, heads_acc, o, l = seen[i]
        qh = util.to_np(q).reshape(1, heads, 128)
        want = ref.attention(pool, util.to_np(table), [i + 1], [1], qh, SCALE)
        assert np.all(np.abs(util.to_np(heads_acc) - want[0]) <= want[2])
        o2 = torch.empty_like(o)
        ops.gemv_attn_heads_f32_w4a16(*W["o"], heads_acc, before, o2, H, H)
        assert torch.equal(o, o2)
    rel = 0.0
    for i in range(steps):
        add, r = ref.key_weights(pool, util.to_np(table), [i + 1], [1], util.to_np(seen[i][1]).reshape(1, heads, 128), util.to_np(seen[i][4]).astype(np.float64), SCALE)
        total += add
        rel = max(rel, r)
    got = util.to_np(cache.key_weight)
    assert np.all(np.abs(got - total) <= total * (2 * rel + steps * 2.0 ** -24))
    dst, new_lens, kept = i32(np.array([[6, 4]])), i32([0]), i32(np.zeros((1, kv, 20)))
    ops.kv4_evict(cache, batch, dst, new_lens, kept, 2, 20, 2, 6)
    after = ops.KV4Batch.of(dst, new_lens)
    ops.attention_kv4(cache, after, bufs["q"], acc, lse, ws, heads, n, True, SCALE)
    pool.words[:] = words_of(cache)
    want = ref.attention(pool, np.array([[6, 4]]), [20], [1], util.to_np(bufs["q"]).reshape(1, heads, 128), SCALE)
    assert np.all(np.abs(util.to_np(acc) - want[0]) <= want[2])
    for h_ in range(kv):
        assert util.to_np(kept)[0, h_].tolist() == ref.evict(got, util.to_np(table)[0], steps, h_, page, 2 * per, 20, 2, 6)


@pytest.mark.parametrize("tokens,f32", [(3, True), (60, False)])
def test_rows_behind_the_last_sequence_are_left_alone(ops, tokens, f32):
    lens, new, kv, heads, page = [70, 30], [tokens, 5], 2, 8, 16
    rng, pool, table, cache, batch = make(ops, 11, lens, new, kv, page)
    T = sum(new)
    batch.num_tokens = T + 9
    q = np.full((T + 9, heads, 128), np.nan, BF)
    q[:T] = rng.standard_normal((T, heads, 128))
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, f32)
    few = few_rows(batch, heads, cache, f32)
    check_attention(np.concatenate([got[:T], got[-1:]]), np.concatenate([lse[:T], lse[-1:]]), ref.attention(pool, table, lens, new, q[:T], SCALE, not few), T, f32)
    assert (got[T:] == 7).all() and (lse[T:] == 7).all()
    before = util.to_np(cache.key_weight).copy()
    ops.kv4_add_key_weights(cache, batch, util.to_dev(q), util.to_dev(lse), heads, SCALE)
    add, rel = ref.key_weights(pool, table, lens, new, q[:T], lse[:T].astype(np.float64), SCALE)
    after = util.to_np(cache.key_weight)
    assert np.all(np.abs(after - before - add) <= add * 2 * rel + np.abs(after) * 2.0 ** -22)


@pytest.mark.parametrize("rows", [63, 64, 65])
def test_both_sides_of_the_border_between_the_forms(ops, rows):
    """One key/value head and one query head a sequence: a token is a row."""
    lens, new, kv, heads, page = [300], [rows], 1, 1, 16
    rng, pool, table, cache, batch = make(ops, 12, lens, new, kv, page)
    q = rng.standard_normal((rows, heads, 128)).astype(BF)
    got, lse = attend(ops, cache, batch, util.to_dev(q), heads, False)
    check_attention(got, lse, ref.attention(pool, table, lens, new, q, SCALE, rows >= 64), rows, False)


@pytest.mark.parametrize("lens,new,kv,heads,f32", [([900, 40], [1, 1], 2, 12, True), ([900, 40], [1, 1], 2, 12, False), ([900, 400], [5, 4], 2, 12, True),
                                                   ([900, 400], [200, 100], 2, 12, False)])
def test_the_same_call_gives_the_same_bits(ops, lens, new, kv, heads, f32):
    """Twice, with programmatic dependent launch off, and out of a graph that is replayed after the lengths have changed and come back."""
    rng, pool, table, cache, batch = make(ops, 13, lens, new, kv, 16)
    T = sum(new)
    q = util.to_dev(rng.standard_normal((T, heads, 128)).astype(BF))
    first = attend(ops, cache, batch, q, heads, f32)
    again = attend(ops, cache, batch, q, heads, f32)
    ops.set_pdl(False)
    try:
        plain = attend(ops, cache, batch, q, heads, f32)
    finally:
        ops.set_pdl(True)
    for other in (again, plain):
        assert np.array_equal(first[0], other[0]) and np.array_equal(first[1], other[1])
    out = torch.empty(T, heads, 128, dtype=torch.float32 if f32 else torch.float16, device="cuda")
    lse = torch.empty(T, heads, device="cuda")
    n = ops.attention_kv4_workspace_bytes(T, len(lens), heads, kv)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.attention_kv4(cache, batch, q, out, lse, ws, heads, n, f32, SCALE)
        ops.kv4_add_key_weights(cache, batch, q, lse, heads, SCALE)
    short = [max(L // 3, k) for L, k in zip(lens, new)]
    batch.seq_lens.copy_(i32(short))
    graph.replay()
    want = ref.attention(pool, table, short, new, util.to_np(q), SCALE, not few_rows(batch, heads, cache, f32))
    check_attention(np.concatenate([util.to_np(out), np.full((1, heads, 128), 7)]), np.concatenate([util.to_np(lse), np.full((1, heads), 7.0)]), want, T, f32)
    batch.seq_lens.copy_(i32(lens))
    graph.replay()
    assert np.array_equal(util.to_np(out), first[0][:T]) and np.array_equal(util.to_np(lse), first[1][:T])


def test_two_streams_with_a_workspace_each(ops):
    lens, kv, heads = [3000], 2, 12
    rng, pool, table, cache, batch = make(ops, 14, lens, [1], kv, 64)
    chunk = ops.KV4Batch.of(batch.block_table, batch.seq_lens, i32([0, 300]), 300)
    q1, q2 = (util.to_dev(rng.standard_normal((n, heads, 128)).astype(BF)) for n in (1, 300))
    want1, want2 = attend(ops, cache, batch, q1, heads, True)[0], attend(ops, cache, chunk, q2, heads, False)[0]
    n1, n2 = ops.attention_kv4_workspace_bytes(1, 1, heads, kv), ops.attention_kv4_workspace_bytes(300, 1, heads, kv)
    w1, w2 = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (n1, n2))
    o1, o2 = torch.empty(1, heads, 128, device="cuda"), torch.empty(300, heads, 128, dtype=torch.float16, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        ops.attention_kv4(cache, batch, q1, o1, None, w1, heads, n1, True, SCALE, stream=s1)
        ops.attention_kv4(cache, chunk, q2, o2, None, w2, heads, n2, False, SCALE, stream=s2)
    torch.cuda.synchronize()
    assert np.array_equal(util.to_np(o1)[0], want1[0]) and np.array_equal(util.to_np(o2), want2[:300])


def test_a_pool_of_more_than_4_gib(ops):
    """The same sequences on the last pages of a pool whose offsets pass 32 bits: the same bits from every operator."""
    lens, new, kv, heads, page = [500, 130], [70, 64], 2, 8, 64
    rng, pool, table, small, batch = make(ops, 15, lens, new, kv, page)
    n = pool.num_pages
    record = kv * 34 * page * 4
    big_n = (4 << 30) // record + 2 * n
    pages = torch.zeros(big_n, kv, 34 * page, dtype=torch.int32, device="cuda")
    assert (big_n - n) * record > 1 << 32
    pages[-n:] = small.pages
    weight = torch.zeros(big_n, kv, page, device="cuda")
    weight[-n:] = small.key_weight
    big = ops.KV4Cache(pages, weight, big_n, kv, page)
    moved = ops.KV4Batch.of(batch.block_table + (big_n - n), batch.seq_lens, batch.query_start, batch.num_tokens)
    T = sum(new)
    q, k, v = (util.to_dev(rng.standard_normal((T, w * 128)).astype(BF)) for w in (heads, kv, kv))
    results = []
    for cache, b in ((small, batch), (big, moved)):
        ops.kv4_append(cache, b, None, k, v, None, None, None, None, None, None, heads)
        kr, vr = (torch.empty(T, kv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
        ops.kv4_read(cache, b, kr, vr)
        out = [kr.clone(), vr.clone(), cache.pages[-n:].clone()]
        for f32 in (True, False):
            o, l = attend(ops, cache, b, q, heads, f32)
            out += [torch.from_numpy(o), torch.from_numpy(l)]
        lse = util.to_dev(l[:T])
        ops.kv4_add_key_weights(cache, b, q, lse, heads, SCALE)
        out.append(cache.key_weight[-n:].clone())
        spare = [p for p in range(n) if p not in set(table.reshape(-1).tolist())]
        dst = i32([[spare[0] + cache.num_pages - n], [spare[1] + cache.num_pages - n]])
        kept, new_lens = i32(np.zeros((2, kv, 40))), i32([0, 0])
        ops.kv4_evict(cache, b, dst, new_lens, kept, 1, 40, 4, 8)
        out += [kept, new_lens, cache.pages[-n:].clone(), cache.key_weight[-n:].clone()]
        results.append([util.to_np(t) for t in out])
    for a, b in zip(*results):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")


def test_waits_of_the_chunk_form_did_not_run_out(ops):
    assert ops.debug_counter(0) == 0


# ---- the decode sweep with caches ----------------------------------------------------------------------------------------


def sweep_case(ops, layers, heads, kv, page, length, flags, weights, seed=5):
    """A small model with a cache of `length` positions a layer; everything a sweep and a sequence of separate calls need."""
    from qwen_engine_b200 import synth
    H, inter, qd, kd = 512, 1024, 128 * heads, 128 * kv
    rng = np.random.default_rng(seed)
    per = -(-(length + 8) // page)
    table, lens = i32(rng.permutation(per + 2)[None, :per].copy()), i32([length])
    L, caches, biases, words = [], [], [], []
    for l in range(layers):
        d = {n: (util.to_dev(synth.packed_weights(seed, f"{n}{l}", r, c)), util.to_dev(synth.scales(seed, f"{n}{l}", r, c)))
             for n, r, c in (("q", qd, H), ("k", kd, H), ("v", kd, H), ("o", H, qd), ("gate_up", 2 * inter, H), ("down", H, inter))}
        d["input_norm"] = d["post_norm"] = torch.full((H,), 0.05, dtype=torch.float16, device="cuda")
        L.append(d)
        pool = ref.Pool(per + 2, kv, page).fill_random(rng, 1.5, 0.7)
        words.append(pool.words.copy())
        caches.append(ops.KV4Cache(util.to_dev(pool.words), torch.zeros(per + 2, kv, page, device="cuda") if weights else None, per + 2, kv, page))
        biases.append(tuple(util.to_dev(rng.standard_normal(n).astype(BF)) for n in (qd, kd, kd)) if l != 1 else None)
    inv = torch.tensor(1e6 ** (-np.arange(64) / 64), dtype=torch.float32, device="cuda")
    position = i32([length + 100])
    cache = ops.SweepCache(caches, ops.KV4Batch.of(table, lens), SCALE, biases, position, inv, weights)
    sweep = ops.DecodeSweep(L, hidden=H, inter=inter, num_q_heads=heads, num_kv_heads=kv, flags=flags, kv4=cache)
    return H, inter, L, cache, sweep, words


def separate_calls(ops, H, inter, L, cache, heads, h):
    qd, kd = 128 * heads, 128 * cache.caches[0].num_kv_heads
    f16 = lambda n: torch.empty(n, dtype=torch.float16, device="cuda")  # noqa: E731
    n = ops.attention_kv4_workspace_bytes(1, 1, heads, kd // 128)
    ws, acc, lse = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty(heads, 128, device="cuda"), torch.empty(heads, device="cuda")
    for d, c, b in zip(L, cache.caches, cache.biases):
        q, k, v, o, mlp, out = f16(qd), f16(kd), f16(kd), f16(H), f16(inter), f16(H)
        view = ops.QKVProjectionView(*d["q"], q, *d["k"], k, *d["v"], v)
        ops.launch_gemv_qkv_rmsnorm_w4a16(view, h, d["input_norm"], in_features=H, num_q_heads=heads, num_kv_heads=kd // 128)
        ops.kv4_append(c, cache.batch, q, k, v, *(b or (None,) * 3), cache.position, cache.rope_inv_freq, q, heads)
        ops.attention_kv4(c, cache.batch, q, acc, lse, ws, heads, n, True, SCALE)
        if cache.add_key_weights:
            ops.kv4_add_key_weights(c, cache.batch, q, lse, heads, SCALE)
        ops.gemv_attn_heads_f32_w4a16(*d["o"], acc, h, o, H, qd)
        ops.launch_gemv_dual_gate_up_swiglu_rmsnorm_w4a16(*d["gate_up"], o, d["post_norm"], mlp, H, inter)
        ops.launch_gemv_w4a16(*d["down"], mlp, o, out, H, inter)
        h = out
    return h


@pytest.mark.parametrize("flags", ["SWEEP_DEFAULT", "SWEEP_SEPARATE", "SWEEP_FUSE_ALL", "SWEEP_PUBLISH_AMAX"])
@pytest.mark.parametrize("heads,kv,page,length,weights", [(12, 2, 16, 0, True), (4, 1, 32, 20, False), (8, 8, 16, 700, True)])
def test_decode_sweep_with_caches_is_the_separate_calls(ops, heads, kv, page, length, weights, flags):
    """Six steps on a growing sequence: hidden state, pages and weights bit for bit; making the sweep stores nothing."""
    H, inter, L, cache, sweep, words = sweep_case(ops, 3, heads, kv, page, length, getattr(ops, flags), weights)
    first = [c.pages.clone() for c in cache.caches]
    other = ops.SweepCache([ops.KV4Cache(c.pages.clone(), None if c.key_weight is None else c.key_weight.clone(), c.num_pages, kv, page) for c in cache.caches],
                           cache.batch, SCALE, cache.biases, cache.position, cache.rope_inv_freq, weights)
    torch.cuda.synchronize()
    assert all(np.array_equal(words_of(c), w) and (not weights or not c.key_weight.any()) for c, w in zip(cache.caches, words))
    h = util.to_dev(np.random.default_rng(3).standard_normal(H).astype(BF))
    for step in range(6):
        cache.batch.seq_lens.add_(1)
        cache.position.add_(1)
        out = torch.empty_like(h)
        sweep.run_device(h, out)
        want = separate_calls(ops, H, inter, L, other, heads, h)
        assert torch.equal(out, want), step
        assert torch.isfinite(out).all()
        for a, b, f in zip(cache.caches, other.caches, first):
            assert torch.equal(a.pages, b.pages) and not torch.equal(a.pages, f)
            if weights:
                assert torch.equal(a.key_weight, b.key_weight) and a.key_weight.sum().item() > 0
        h = out
    sweep.close()


def test_two_sweeps_from_one_cache_object_keep_their_workspaces(ops):
    """Two graphs made from one SweepCache, run in turn, give what each gives alone."""
    H, inter, L, cache, one, _ = sweep_case(ops, 2, 4, 2, 16, 40, ops.SWEEP_DEFAULT, False)
    two = ops.DecodeSweep(L, hidden=H, inter=inter, num_q_heads=4, num_kv_heads=2, kv4=cache)
    cache.batch.seq_lens.add_(1)
    h = util.to_dev(np.random.default_rng(3).standard_normal(H).astype(BF))
    a, b, c = (torch.empty_like(h) for _ in range(3))
    one.run_device(h, a)
    two.run_device(h, b)
    one.run_device(h, c)
    assert torch.equal(a, b) and torch.equal(a, c)
    # 3 launches a layer more than the sweep without caches: append, attention, its join
    plain = ops.DecodeSweep(L, hidden=H, inter=inter, num_q_heads=4, num_kv_heads=2)
    assert one.launches == plain.launches + 2 * 3


def test_key_weights_of_pages_that_sequences_share(ops):
    """Forty sequences over one prefix (their tables begin with the same pages): a position's weight is the sum over all of them.
    Every addition may be off by half a step of the total on top of what each sequence's own sum may be off."""
    seqs, kv, heads, page, shared = 40, 2, 4, 16, 6
    lens = [page * shared + 3 + b % 11 for b in range(seqs)]
    rng, pool, table, cache, batch = make(ops, 21, lens, [1] * seqs, kv, page)
    table[:, :shared] = table[0, :shared]
    batch = ops.KV4Batch.of(i32(table), batch.seq_lens)
    q = (1.2 * rng.standard_normal((seqs, heads, 128))).astype(BF)
    lse = ref.attention(pool, table, lens, [1] * seqs, q, SCALE)[1].astype(np.float32)
    add, rel = ref.key_weights(pool, table, lens, [1] * seqs, q, lse.astype(np.float64), SCALE)
    ops.kv4_add_key_weights(cache, batch, util.to_dev(q), util.to_dev(lse), heads, SCALE)
    want = pool.weight + add
    got = util.to_np(cache.key_weight)
    assert np.all(np.abs(got - want) <= add * rel + seqs * np.abs(want) * 2.0 ** -24)
    assert np.array_equal(got[add == 0], pool.weight[add == 0])


def test_decode_sweep_goes_on_after_an_eviction(ops):
    """Three steps, every layer's cache cut to 16 positions on a fresh page, table and lengths copied into the sweep's arrays, three more
    steps: hidden state, pages and weights as the separate calls leave them."""
    heads, kv, page, length = 4, 1, 32, 20
    H, inter, L, cache, sweep, _ = sweep_case(ops, 3, heads, kv, page, length, ops.SWEEP_DEFAULT, True)
    other = ops.SweepCache([ops.KV4Cache(c.pages.clone(), c.key_weight.clone(), c.num_pages, kv, page) for c in cache.caches],
                           cache.batch, SCALE, cache.biases, cache.position, cache.rope_inv_freq, True)
    h = util.to_dev(np.random.default_rng(4).standard_normal(H).astype(BF))
    table, lens = cache.batch.block_table, cache.batch.seq_lens
    for step in range(6):
        if step == 3:
            fresh = i32([[next(p for p in range(3) if p != table.item())]])
            new_lens, kept = i32([0]), i32(np.zeros((1, kv, 16)))
            for c in cache.caches + other.caches:
                ops.kv4_evict(c, cache.batch, fresh, new_lens, kept, 1, 16, 4, 6)
            table.copy_(fresh), lens.copy_(new_lens)
            assert lens.item() == 16
        lens.add_(1)
        cache.position.add_(1)
        out = torch.empty_like(h)
        sweep.run_device(h, out)
        assert torch.equal(out, separate_calls(ops, H, inter, L, other, heads, h)) and torch.isfinite(out).all(), step
        for a, b in zip(cache.caches, other.caches):
            assert torch.equal(a.pages, b.pages) and torch.equal(a.key_weight, b.key_weight), step
        h = out
    sweep.close()
