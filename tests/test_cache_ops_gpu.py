"""The 8-bit paged key/value cache and attention over it (mb_op_cache_*)
against plain float64 forms.

Writing and reading: scales are powers of two, so every code is determined
and the values read back must be equal bit for bit.

Attention, from its arithmetic: with S = scale |q|_2 |k|_2 a score is off by at
most S (2^-21 for the two-part queries, 2^-20 for its sums), a probability by
that and 2^-21, an output by twice a probability's share of the largest |v|:
4e-6 (1 + S) max|v| in single precision.  16-bit outputs add their own half
unit (2^-11, 2^-8 of the value) and the probabilities' one 11-bit rounding,
2^-11 max|v|.  The base-2 log-sum-exp is off by log2(e) times a score's error
and its own rounding."""

import math

import numpy as np
import pytest

from grokking_abmod_b200 import MeshError, UnsupportedShape, ops

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


DTYPES = ("float32", "bfloat16", "float16")


def _pow2_scale(amax):
    """Smallest 2^e >= 2^-126 with amax <= 127 2^e."""
    if not math.isfinite(amax):
        return math.nan
    e = -126
    if amax > 0:
        m, x = math.frexp(amax / 127.0)
        e = max(e, x - 1 if m == 0.5 else x)
    return math.ldexp(1.0, e)


class Plain:
    """The cache as float64 arithmetic on the host, page by page."""

    def __init__(self, pages, heads, tokens, head_dim):
        self.codes = np.zeros((2, pages, heads, tokens, head_dim))
        self.scale = np.zeros((2, pages, heads))
        self.tokens = tokens

    def write(self, kv, table, lengths, news):
        row = 0
        for b, (n, m) in enumerate(zip(lengths, news)):
            old = n - m
            for i in range(old // self.tokens, -(-n // self.tokens)):
                lo, hi = i * self.tokens, min(n, (i + 1) * self.tokens)
                start = max(lo, old)
                if hi <= start:
                    continue
                page = table[b][i]
                for w in range(2):
                    for h in range(kv[w].shape[1]):
                        x = kv[w][row + start - old:row + hi - old, h]
                        s = _pow2_scale(np.abs(x).max() if np.isfinite(x).all() else np.inf)
                        c = self.codes[w, page, h]
                        if start > lo:
                            was = self.scale[w, page, h]
                            s = was if math.isnan(was) or was > s else s
                            if s != was and not math.isnan(was):
                                c[:start - lo] = np.rint(c[:start - lo] * (was / s))
                        with np.errstate(invalid="ignore"):
                            c[start - lo:hi - lo] = 0 if math.isnan(s) else np.rint(x / s)
                        self.scale[w, page, h] = s
            row += m

    def read(self, w, table_row, n):
        out = [self.codes[w, table_row[p // self.tokens], :, p % self.tokens]
               * self.scale[w, table_row[p // self.tokens]][:, None] for p in range(n)]
        return np.stack(out) if out else np.zeros((0,) + self.codes.shape[2:3] + self.codes.shape[4:])


def _table(rng, lengths, tokens, spare=2):
    per = [-(-n // tokens) for n in lengths]
    order = rng.permutation(sum(per) + spare)
    table = np.full((len(lengths), max(per + [1])), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(per) + spare


def _i32(a):
    torch = _torch()
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _rows(rng, shape, dtype, scale=1.0):
    """Values that the type holds, as (float64 array, CUDA tensor)."""
    torch = _torch()
    t = torch.from_numpy(rng.normal(0, scale, shape).astype(np.float32)).to(getattr(torch, dtype))
    return t.double().numpy(), t.cuda()


def _offsets(news):
    return np.concatenate([[0], np.cumsum(news)])


def _read_all(cache, table, lengths, head_dim, dtype="float32"):
    torch = _torch()
    k, v = ops.cache_read(cache, _i32(table), _i32(lengths), max(max(lengths), 1), head_dim=head_dim,
                          dtype=getattr(torch, dtype))
    return k.double().cpu().numpy(), v.double().cpu().numpy()


def _equal(plain, cache, table, lengths, head_dim, dtype="float32"):
    got = _read_all(cache, table, lengths, head_dim, dtype)
    for w in range(2):
        for b, n in enumerate(lengths):
            np.testing.assert_array_equal(got[w][b, :n], plain.read(w, table[b], n))
            assert not got[w][b, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,head_dim,tokens", [(8, 64, 16), (3, 80, 32), (1, 128, 128), (2, 7, 64), (5, 1, 16),
                                                  (4, 96, 64), (16, 30, 32)])
def test_written_rows_read_back_exactly(dtype, heads, head_dim, tokens):
    """Prompts, single tokens and nothing, in turn, into the same pages; a
    later token with larger values moves the page's scale."""
    rng = np.random.default_rng(heads * head_dim + tokens)
    steps = [[tokens + 5, 0, 1, 2 * tokens], [1, 1, 1, 1], [3, tokens, 0, 1], [1, 1, 1, 1], [0, tokens - 1, 200, 1]]
    final = np.sum(steps, axis=0)
    table, pages = _table(rng, final, tokens)
    plain = Plain(pages, heads, tokens, head_dim)
    cache = ops.new_kv_cache(pages, heads, head_dim, tokens)
    for t in cache[2:]:
        t.fill_(float("nan"))  # what was there before is of no account
    status = ops.new_status()
    lengths = np.zeros(4, dtype=np.int64)
    for i, news in enumerate(steps):
        lengths = lengths + news
        (k64, k), (v64, v) = (_rows(rng, (sum(news), heads, head_dim), dtype, 2.0 ** (2 * i)) for _ in range(2))
        plain.write((k64, v64), table, lengths, news)
        ops.cache_write(cache, k, v, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=max(news),
                        status=status)
        ops.check_status(status)
        _equal(plain, cache, table, lengths, head_dim)
    assert not cache.k[..., head_dim:].any() and not cache.v[..., head_dim:].any()


def test_one_row_each_and_strided_rows():
    """No offsets; K and V as slices of a fused projection, heads before rows."""
    torch = _torch()
    rng = np.random.default_rng(4)
    batch, heads, hd, tokens = 37, 4, 24, 16
    lengths = rng.integers(1, 60, batch)
    table, pages = _table(rng, lengths, tokens)
    plain, cache = Plain(pages, heads, tokens, hd), ops.new_kv_cache(pages, heads, hd, tokens)
    fused = torch.from_numpy(rng.normal(0, 1, (batch, 3 * heads * hd + 1)).astype(np.float32)).cuda()
    k = fused[:, 1:1 + heads * hd].unflatten(1, (heads, hd))
    v = torch.from_numpy(rng.normal(0, 1, (heads, batch, hd)).astype(np.float32)).cuda().transpose(0, 1)
    first = np.maximum(lengths - 1, 0)
    # what stands before the new token
    k0, v0 = (rng.normal(0, 1, (first.sum(), heads, hd)).astype(np.float32) for _ in range(2))
    plain.write((k0.astype(np.float64), v0.astype(np.float64)), table, first, first)
    ops.cache_write(cache, torch.from_numpy(k0).cuda(), torch.from_numpy(v0).cuda(), _i32(table), _i32(first),
                    _i32(_offsets(first)))
    plain.write((k.double().cpu().numpy(), v.double().cpu().numpy()), table, lengths, [1] * batch)
    ops.cache_write(cache, k, v, _i32(table), _i32(lengths))
    _equal(plain, cache, table, lengths, hd)
    # a window of it, from each sequence's own position, in 16 bits
    start = rng.integers(-3, 60, batch)
    got = ops.cache_read(cache, _i32(table), _i32(lengths), 9, first=_i32(start), head_dim=hd, dtype=torch.bfloat16)
    for w in range(2):
        values = got[w].double().cpu().numpy()
        for b in range(batch):
            for i in range(9):
                p = start[b] + i
                want = plain.read(w, table[b], lengths[b])[p] if 0 <= p < lengths[b] else 0.0
                np.testing.assert_array_equal(values[b, i], np.broadcast_to(want, values[b, i].shape))


def test_extreme_values():
    """Zeros, the smallest and largest numbers, exact powers, infinities and
    NaN: those spoil their own page and head only, until it is begun again."""
    torch = _torch()
    tokens, hd = 16, 32
    heads = 10
    x = np.zeros((tokens, heads, hd))
    x[:, 1] = 1e-45
    x[:, 2] = 3e38
    x[3, 3, 5] = 127.0
    x[3, 4, 5] = np.nextafter(np.float32(127.0), np.float32(200))
    x[:, 5] = np.ldexp(1.0, np.arange(-100, -100 + hd))
    x[2, 6, 1] = np.inf
    x[9, 7, 0] = np.nan
    x[9, 8, 0] = -np.inf
    x[:, 9] = np.linspace(-1, 1, hd)
    x = x.astype(np.float32).astype(np.float64)
    table, lengths = np.array([[1]], np.int32), [tokens]
    plain, cache = Plain(2, heads, tokens, hd), ops.new_kv_cache(2, heads, hd, tokens)
    t = torch.from_numpy(x.astype(np.float32)).cuda()
    for kv in (t, torch.ones_like(t)):
        plain.write((kv.double().cpu().numpy(),) * 2, table, lengths, lengths)
        ops.cache_write(cache, kv, kv, _i32(table), _i32(lengths), _i32([0, tokens]))
        _equal(plain, cache, table, lengths, hd)


def test_what_does_not_fit_is_skipped_and_reported():
    torch = _torch()
    heads, hd, tokens = 2, 32, 16
    cache = ops.new_kv_cache(3, heads, hd, tokens)
    ones = torch.ones((2, heads, hd), device="cuda")

    def code(f):
        status = ops.new_status()
        f(status)
        return int(status.item())

    table = _i32([[0], [1]])
    assert code(lambda s: ops.cache_write(cache, ones, ones, table, _i32([1, 16]), status=s)) == 0
    before = [t.clone() for t in cache]
    assert code(lambda s: ops.cache_write(cache, ones * 9, ones, _i32([[3], [-1]]), _i32([1, 16]), status=s)) == 2
    assert code(lambda s: ops.cache_write(cache, ones * 9, ones, table, _i32([0, 17]), status=s)) == 4
    assert code(lambda s: ops.cache_write(cache, ones * 9, ones, table, _i32([1, 1]), _i32([0, 9, 2]), max_new=9,
                                          status=s)) == 8
    for was, now in zip(before, cache):
        assert torch.equal(was, now)
    assert code(lambda s: ops.cache_read(cache, _i32([[0], [7]]), _i32([1, 1]), 1, status=s)) == 2
    assert code(lambda s: ops.cache_read(cache, table, _i32([1, 17]), 1, status=s)) == 4
    q = torch.ones((2, heads, hd), device="cuda")
    for lengths, offsets, pages, want in (([1, 17], None, [[0], [1]], 4), ([0, 1], None, [[0], [1]], 4),
                                          ([1, 1], [0, 1, 3], [[0], [1]], 8), ([1, 1], None, [[0], [5]], 2)):
        status = ops.new_status()
        out, lse = ops.cache_attention(q, cache, _i32(pages), _i32(lengths),
                                       _i32(offsets) if offsets is not None else None, max_new=2, status=status)
        assert int(status.item()) == want
        bad = 0 if lengths[0] == 0 else 1
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[:, bad]).all()
        assert torch.isfinite(out[1 - bad]).all()
    # more new rows than announced: the ones past them are NaN
    q = torch.ones((12, heads, hd), device="cuda")
    status = ops.new_status()
    out, _ = ops.cache_attention(q, cache, _i32([[0]]), _i32([16]), _i32([0, 12]), max_new=1, status=status)
    assert int(status.item()) == 8 and torch.isnan(out[-1]).all() and torch.isfinite(out[0]).all()


# ---------------------------------------------------------------- attention
def _filled(rng, lengths, heads, hd, tokens, spread=0.0):
    """A cache of random codes and scales, its float64 values, and its table;
    scales of pages in no sequence are NaN."""
    torch = _torch()
    table, pages = _table(rng, lengths, tokens)
    width = -(-hd // 32) * 32
    codes = np.clip(np.rint(rng.normal(0, 40, (2, pages, heads, tokens, width))), -127, 127)
    codes[..., hd:] = 0
    scale = np.ldexp(1.0, rng.integers(-6, -3, (2, pages, heads)) + np.rint(rng.normal(0, spread, (2, pages, heads))).astype(int))
    unused = np.setdiff1d(np.arange(pages), table[table >= 0])
    values = codes * scale[..., None, None]
    poisoned = scale.copy()
    poisoned[:, unused] = np.nan
    cache = ops.KvCache(*(torch.from_numpy(c.astype(np.int8)).cuda() for c in codes),
                        *(torch.from_numpy(s.astype(np.float32)).cuda() for s in poisoned))
    return cache, values[..., :hd], table


def _attend(q, values, table, lengths, news, first, tokens, scale):
    """(out, lse2) in float64, and S and max|v| for the bound."""
    rows, heads, hd = q.shape
    kv_heads = values.shape[2]
    group = heads // kv_heads
    out, lse = np.zeros_like(q), np.full((heads, rows), -np.inf)
    s_bound = 0.0
    row = 0
    for b, (n, m) in enumerate(zip(lengths, news)):
        pages = table[b, :-(-n // tokens)]
        k, v = (values[w, pages].transpose(1, 0, 2, 3).reshape(kv_heads, -1, hd)[:, :n] for w in range(2))
        for i in range(m):
            lo, hi = max(0, first[b]), n - m + i + 1
            if lo < hi:
                for a in range(heads):
                    s = scale * (k[a // group, lo:hi] @ q[row, a])
                    s_bound = max(s_bound, abs(scale) * np.linalg.norm(q[row, a])
                                  * np.linalg.norm(k[a // group, lo:hi], axis=1).max())
                    p = np.exp(s - s.max())
                    out[row, a] = p @ v[a // group, lo:hi] / p.sum()
                    lse[a, row] = (s.max() + math.log(p.sum())) / math.log(2)
            row += 1
    return out, lse, s_bound


def _check(q64, q, cache, values, table, lengths, news, tokens, first=None, scale=None, offsets=True, dtype="float32",
           max_tokens=None):
    hd = q64.shape[2]
    status = ops.new_status()
    out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)) if offsets else None,
                                   first=_i32(first) if first is not None else None, scale=scale,
                                   max_new=max(max(news), 1) if offsets else None,
                                   max_tokens=max(lengths) if max_tokens is None else max_tokens, status=status)
    ops.check_status(status)
    want, want_lse, s = _attend(q64, values, table, lengths, news, first if first is not None else [0] * len(lengths),
                                tokens, 1 / math.sqrt(hd) if scale is None else scale)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    vmax = np.abs(values[1]).max()
    tol = 4e-6 * (1 + s) * vmax
    if dtype != "float32":
        tol += (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11) * np.abs(want) + 2.0 ** -11 * vmax
    assert out.dtype == q.dtype and np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()
    empty = np.isneginf(want_lse)
    assert np.array_equal(empty, np.isneginf(got_lse))
    assert np.all(np.abs(got_lse - want_lse)[~empty] <= 4e-6 * (1 + s) * 1.4427 + 2.0 ** -22 * np.abs(want_lse[~empty]))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,group,hd,tokens", [(8, 1, 64, 16), (2, 4, 128, 64), (1, 8, 96, 32), (3, 1, 32, 128),
                                                      (2, 3, 80, 16), (1, 16, 16, 32), (2, 12, 128, 16), (4, 2, 2, 64),
                                                      (1, 1, 1, 16), (2, 5, 127, 32)])
def test_single_tokens(dtype, kv_heads, group, hd, tokens):
    rng = np.random.default_rng(hd * group + tokens)
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 100, 129, 257, 700]
    cache, values, table = _filled(rng, lengths, kv_heads, hd, tokens)
    q64, q = _rows(rng, (len(lengths), kv_heads * group, hd), dtype, 1.5)
    _check(q64, q, cache, values, table, lengths, [1] * len(lengths), tokens, offsets=False, dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,group,hd,tokens", [(2, 1, 64, 16), (1, 4, 128, 64), (2, 2, 96, 32), (1, 1, 32, 128),
                                                      (1, 3, 80, 16), (2, 1, 17, 32)])
def test_prompts_of_unequal_lengths(dtype, kv_heads, group, hd, tokens):
    """Whole prompts, parts behind a filled cache, single rows and none."""
    rng = np.random.default_rng(hd + group)
    news = [130, 1, 0, 65, 257, 3, 128]
    lengths = [130, 500, 40, 65 + 333, 257, 5, 128 + 1]
    cache, values, table = _filled(rng, lengths, kv_heads, hd, tokens)
    q64, q = _rows(rng, (sum(news), kv_heads * group, hd), dtype)
    _check(q64, q, cache, values, table, lengths, news, tokens, dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,group,hd,tokens", [(2, 1, 64, 16), (1, 3, 128, 64), (1, 2, 90, 32)])
def test_one_prompt_among_single_tokens(dtype, kv_heads, group, hd, tokens):
    """Few rows on average, many in one sequence."""
    rng = np.random.default_rng(hd + group)
    news = [1, 0, 1, 70, 1, 1, 2, 1, 1, 1, 1, 1]
    lengths = [n + 37 * i for i, n in enumerate(news)]
    cache, values, table = _filled(rng, lengths, kv_heads, hd, tokens)
    q64, q = _rows(rng, (sum(news), kv_heads * group, hd), dtype)
    _check(q64, q, cache, values, table, lengths, news, tokens, dtype=dtype)


@pytest.mark.parametrize("news,hd,tokens", [([1, 1, 1, 1, 1, 1], 64, 16), ([40, 33, 150, 1, 7, 200], 64, 32),
                                            ([150, 2, 129, 130, 31, 9], 128, 16)])
def test_left_limits_and_rows_that_see_nothing(news, hd, tokens):
    """first inside, at and past the length, negative, and between new rows:
    the earlier ones see nothing."""
    rng = np.random.default_rng(hd + len(news))
    lengths = [n + 90 for n in news]
    first = [0, 47, lengths[2], lengths[3] - 1, -5, lengths[5] - 4]
    cache, values, table = _filled(rng, lengths, 2, hd, tokens)
    for b, f in enumerate(first):  # pages before it may be gone
        table[b, :max(0, min(f, lengths[b])) // tokens] = 10 ** 6
    held = np.where(table == 10 ** 6, 0, table)
    q64, q = _rows(rng, (sum(news), 4, hd), "float32")
    status = ops.new_status()
    out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), first=_i32(first),
                                   max_new=max(news), max_tokens=max(lengths), status=status)
    ops.check_status(status)
    assert _torch().isfinite(out).all()
    _check(q64, q, cache, values, held, lengths, news, tokens, first=first)
    empty = _offsets(news)[2]
    assert not out[empty:empty + news[2]].any() and _torch().isneginf(lse[:, empty:empty + news[2]]).all()


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("max_tokens", [0, 64, 5000, 100000])
def test_any_split_of_a_long_sequence(new, max_tokens):
    """max_tokens below, near and far above the lengths only moves the cuts."""
    rng = np.random.default_rng(new)
    lengths = [5003, 40, 2048]
    cache, values, table = _filled(rng, lengths, 2, 64, 32)
    q64, q = _rows(rng, (3 * new, 4, 64), "float32", 2.0)
    _check(q64, q, cache, values, table, lengths, [new] * 3, 32, max_tokens=max_tokens)


def test_scales_that_differ_widely():
    """Pages of very different magnitude, all-zero pages and a large q."""
    rng = np.random.default_rng(5)
    lengths = [300, 90]
    cache, values, table = _filled(rng, lengths, 2, 64, 16, spread=2.0)
    # zero V pages with the smallest scale
    for page in table[0, 2:5]:
        cache.v[page] = 0
        cache.v_scale[page] = 2.0 ** -126
        values[1, page] = 0
    for news in ([1, 1], [200, 90]):
        q64, q = _rows(rng, (sum(news), 2, 64), "float32", 0.02)
        _check(q64, q, cache, values, table, lengths, news, 16)
        _check(q64 * 2.0 ** 80, q * 2.0 ** 80, cache, values, table, lengths, news, 16, scale=2.0 ** -80)


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 140, 7]])
def test_a_nan_stays_in_its_rows(news):
    torch = _torch()
    rng = np.random.default_rng(6)
    lengths = [200, 150, 40]
    cache, _, table = _filled(rng, lengths, 2, 64, 32)
    _, q = _rows(rng, (sum(news), 2, 64), "float32")
    clean, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=max(news))
    q[0, 1, 3] = float("nan")
    q[1, 0, 0] = float("inf")
    out, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=max(news))
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 1] = bad[1, 0] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
    # a spoilt page: every row that sees it
    cache.v_scale[int(table[2, 0]), 1] = float("nan")
    out, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=max(news))
    assert torch.isnan(out[-1, 1]).all() and torch.isfinite(out[-1, 0]).all()


def test_strided_queries_another_stream_and_repeats():
    """A slice of a fused projection; the same bits on every call."""
    torch = _torch()
    rng = np.random.default_rng(8)
    lengths, news = [300, 260, 17], [5, 130, 17]
    cache, values, table = _filled(rng, lengths, 2, 48, 16)
    fused = torch.from_numpy(rng.normal(0, 1, (sum(news), 3 * 4 * 48 + 3)).astype(np.float32)).cuda()
    q = fused[:, 3 + 48:3 + 5 * 48].unflatten(1, (4, 48))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = _check(q.double().cpu().numpy(), q, cache, values, table, lengths, news, 16)
        again = _check(q.double().cpu().numpy(), q, cache, values, table, lengths, news, 16)
    stream.synchronize()
    assert torch.equal(out, again)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes a tensor: the last pages are reached."""
    torch = _torch()
    heads, hd, tokens = 8, 128, 128
    pages = (1 << 32) // (heads * hd * tokens) + 64
    cache = ops.KvCache(*(torch.empty((pages, heads, tokens, hd), dtype=torch.int8, device="cuda") for _ in range(2)),
                        *(torch.empty((pages, heads), device="cuda") for _ in range(2)))
    rng = np.random.default_rng(9)
    lengths = [200, 70]
    table = np.array([[pages - 1, pages - 2], [3, 0]], np.int32)
    (k64, k), (v64, v) = (_rows(rng, (270, heads, hd), "float32") for _ in range(2))
    ops.cache_write(cache, k, v, _i32(table), _i32(lengths), _i32([0, 200, 270]))
    small = {pages - 1: 0, pages - 2: 1, 3: 2, 0: 3}
    near = np.vectorize(small.get)(table)
    plain = Plain(4, heads, tokens, hd)
    plain.write((k64, v64), near, lengths, lengths)
    got = _read_all(cache, table, lengths, hd)
    values = plain.codes * plain.scale[..., None, None]
    for w in range(2):
        for b, n in enumerate(lengths):
            np.testing.assert_array_equal(got[w][b, :n], plain.read(w, near[b], n))
    for news in ([1, 1], [150, 70]):
        q64, q = _rows(rng, (sum(news), heads, hd), "float32")
        out, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=max(news))
        want, _, s = _attend(q64, values, near, lengths, news, [0, 0], tokens, hd ** -0.5)
        assert np.abs(out.double().cpu().numpy() - want).max() <= 4e-6 * (1 + s) * np.abs(values[1]).max()


def test_refusals():
    torch = _torch()
    cache = ops.new_kv_cache(4, 2, 64, 32)
    q = torch.zeros((2, 4, 64), device="cuda")
    table, lengths = _i32([[0], [1]]), _i32([1, 1])
    call = ops.cache_attention
    with pytest.raises(ValueError):
        call(q.double(), cache, table, lengths)
    with pytest.raises(ValueError):
        call(q.transpose(1, 2), cache, table, lengths)
    with pytest.raises(ValueError):
        call(q, cache, table.long(), lengths)
    with pytest.raises(ValueError):
        call(q, cache, table, lengths[:1])
    with pytest.raises(ValueError):
        call(q, cache._replace(k=cache.k.float()), table, lengths)
    with pytest.raises(ValueError):
        call(q, cache._replace(k_scale=cache.k_scale[:2]), table, lengths)
    with pytest.raises(ValueError):
        call(q.cpu(), cache, table, lengths)
    with pytest.raises(MeshError):
        call(q[:, :3], cache, table, lengths)  # 2 key heads do not divide 3
    with pytest.raises(MeshError):
        call(q[..., :30], cache, table, lengths)  # the cache is 64 wide
    with pytest.raises(MeshError):
        call(q[:1], cache, table, lengths)  # two sequences, one row, no offsets
    with pytest.raises(MeshError):
        call(q, cache, table, lengths, scale=float("inf"))
    with pytest.raises(MeshError):
        call(q, ops.new_kv_cache(4, 2, 64, 48), table, lengths)
    with pytest.raises(UnsupportedShape):
        call(torch.zeros((2, 4, 160), device="cuda"), ops.new_kv_cache(4, 2, 160, 32), table, lengths)
    with pytest.raises(ValueError):
        ops.cache_write(cache, q[:, :2], q[:, :2].half(), table, lengths)
    with pytest.raises(ValueError):
        ops.cache_write(cache, q, q, table, lengths)
    with pytest.raises(ValueError):
        ops.cache_read(cache, table, lengths, 1, dtype=torch.float64)
    # nothing to do is not an error
    none = torch.zeros((0, 4, 64), device="cuda")
    out, lse = call(none, cache, table, lengths, _i32([0, 0, 0]))
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    ops.cache_write(cache, none[:, :2], none[:, :2], table, lengths, _i32([0, 0, 0]))
    assert ops.cache_read(cache, table, lengths, 0)[0].shape == (2, 0, 2, 64)


def test_launches_back_to_back_agree():
    """Prompts whose halves and blocks end on different tiles, many launches in
    a row without waiting: every one the same bits, no wait that gave up."""
    torch = _torch()
    rng = np.random.default_rng(11)
    cases = []
    for hd, dtype in ((64, "float32"), (128, "bfloat16"), (96, "float16"), (128, "float32")):
        news = [300 + 37 * i for i in range(9)]
        lengths = [n + 129 * i for i, n in enumerate(news)]
        cache, _, table = _filled(rng, lengths, 2, hd, 32)
        _, q = _rows(rng, (sum(news), 4, hd), dtype)
        cases.append((q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max(news), max(lengths)))
    status = ops.new_status()
    first, begin = None, torch.cuda.Event(enable_timing=True)
    end = torch.cuda.Event(enable_timing=True)
    for turn in range(60):
        if turn == 1:
            begin.record()
        outs = [ops.cache_attention(q, c, t, n, o, max_new=m, max_tokens=most, status=status)
                for q, c, t, n, o, m, most in cases]
        if first is None:
            first = outs
    end.record()
    ops.check_status(status)
    for a, b in zip(first, outs):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert begin.elapsed_time(end) < 59 * 4 * 50  # a wait that runs out takes about a second


def test_long_prompts_keep_single_precision():
    """Errors of sums over many tiles do not grow with the length: against
    float64 the output stays within twice the error of FP32 arithmetic with
    rounded sums, 2^-24 sqrt(length) of it, and the scores' own 2^-21 S."""
    rng = np.random.default_rng(12)
    for hd, length in ((64, 4096), (128, 3000)):
        cache, values, table = _filled(rng, [length], 1, hd, 64)
        q64, q = _rows(rng, (130, 1, hd), "float32")
        out, _ = ops.cache_attention(q, cache, _i32(table), _i32([length]), _i32([0, 130]), max_new=130)
        want, _, s = _attend(q64, values, table, [length], [130], [0], 64, hd ** -0.5)
        got = out.double().cpu().numpy()
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        # outputs are averages of many values: smaller than them by the effective number of tokens
        shrink = np.sqrt((values[1] ** 2).mean()) / np.sqrt((want ** 2).mean())
        assert rel <= 2 * (2.0 ** -24 * np.sqrt(length) + 2.0 ** -21) * max(1.0, shrink)


@pytest.mark.parametrize("dtype,head_dim,tokens", [("bfloat16", 64, 32), ("float16", 90, 16), ("float32", 64, 16)])
def test_many_pages_in_one_write(dtype, head_dim, tokens):
    """Pages of 129 to 256 vectors, many of them, ragged; then larger values
    into the half-filled ones."""
    rng = np.random.default_rng(head_dim + tokens)
    heads, batch = 8, 16
    steps = [rng.integers(0, 431, batch), rng.integers(1, 431, batch)]
    for news in steps:
        news[3] = 430
    final = np.sum(steps, axis=0)
    table, pages = _table(rng, final, tokens)
    plain, cache = Plain(pages, heads, tokens, head_dim), ops.new_kv_cache(pages, heads, head_dim, tokens)
    status = ops.new_status()
    lengths = np.zeros(batch, dtype=np.int64)
    for i, news in enumerate(steps):
        lengths = lengths + news
        (k64, k), (v64, v) = (_rows(rng, (news.sum(), heads, head_dim), dtype, 2.0 ** (3 * i)) for _ in range(2))
        plain.write((k64, v64), table, lengths, news)
        ops.cache_write(cache, k, v, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=430, status=status)
        ops.check_status(status)
        _equal(plain, cache, table, lengths, head_dim)
