"""What a row of cached attention may depend on: the positions that it sees,
first .. its own, and nothing else, whatever stands beside them in a tile.

A page's scale is NaN once it was given an infinity or a NaN, so spoiling a
scale stands for that.  Tolerances are those of the row's own arithmetic, from
what it sees: with S its largest scale |q|_2 |k|_2, an output is off by
4e-6 (1 + S) of the largest |v| seen; 16-bit outputs add their half unit (2^-11,
2^-8 of the value) and the probabilities' rounding to 11 bits, 2^-11 of the
largest |v| seen.  Weights are kept relative to the largest V scale seen, down
to 2^-36 of it: below the first term."""

import numpy as np
import pytest

from grokking_abmod_b200 import ops
from test_cache_ops_gpu import _filled, _i32, _offsets, _rows, _torch

pytestmark = pytest.mark.gpu

# rows of a few tokens (the split kernel, 8 and 16 rows at once) and prompts (tiles)
FORMS = [("float32", 1, 64, [6, 3]), ("float32", 2, 32, [5, 9]), ("float32", 1, 128, [7, 2]),
         ("bfloat16", 4, 128, [7, 4]), ("float16", 2, 80, [3, 5]), ("bfloat16", 1, 32, [2, 8]),
         ("float32", 1, 64, [150, 90]), ("float32", 2, 96, [333, 64]), ("float32", 1, 128, [270, 70]),
         ("bfloat16", 4, 128, [200, 131]), ("float16", 1, 32, [100, 260])]


def _exact(q, values, table, lengths, news, first, tokens):
    """(out, tolerance of FP32 rows, largest |v| seen) of every row in float64."""
    rows, heads, hd = q.shape
    out, tol, vmax = np.zeros_like(q), np.zeros((rows, heads, 1)), np.zeros((rows, heads, 1))
    group = heads // values.shape[2]
    row = 0
    for b, (n, m) in enumerate(zip(lengths, news)):
        pages = table[b, :-(-n // tokens)]
        k, v = (values[w, pages].transpose(1, 0, 2, 3).reshape(values.shape[2], -1, hd)[:, :n] for w in range(2))
        for i in range(m):
            lo, hi = max(0, first[b]), n - m + i + 1
            for a in range(heads if lo < hi else 0):
                kk, vv = k[a // group, lo:hi], v[a // group, lo:hi]
                s = kk @ q[row, a] / np.sqrt(hd)
                p = np.exp(s - s.max())
                out[row, a] = p @ vv / p.sum()
                big = np.linalg.norm(q[row, a]) * np.linalg.norm(kk, axis=1).max() / np.sqrt(hd)
                vmax[row, a] = np.abs(vv).max()
                tol[row, a] = 4e-6 * (1 + big) * vmax[row, a]
            row += 1
    return out, tol, vmax


def _positions(lengths, news):
    """Each row's own position, and its sequence."""
    return (np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, news)]),
            np.concatenate([np.full(m, b) for b, m in enumerate(news)]))


def _close(got, want, tol, vmax, dtype, keep):
    if dtype != "float32":
        tol = tol + (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11) * np.abs(want) + 2.0 ** -11 * vmax
    over = np.abs(got - want) - tol
    assert np.isfinite(got[keep]).all()
    assert over[keep].max() <= 0, (over / tol)[keep].max()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("tokens", [16, 64])
@pytest.mark.parametrize("dtype,group,hd,news", FORMS)
def test_a_spoilt_page_reaches_the_rows_that_see_it_only(dtype, group, hd, news, tokens, which):
    """Behind a row's own position, and in front of the first one seen."""
    torch = _torch()
    rng = np.random.default_rng(hd + tokens)
    lengths = [news[0] + 75, news[1] + 133]
    first = [0, 100]
    cache, values, table = _filled(rng, lengths, 2, hd, tokens)
    q64, q = _rows(rng, (sum(news), 2 * group, hd), dtype)
    scale = cache.k_scale if which == "k" else cache.v_scale
    # sequence 0: the page of its last new row but one; sequence 1: a page before its first position
    late = (lengths[0] - 2) // tokens
    early = 100 // tokens - 1
    scale[int(table[0, late]), 1] = float("nan")
    scale[int(table[1, early]), 1] = float("nan")
    out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), first=_i32(first),
                                   max_new=max(news), max_tokens=max(lengths))
    want, tol, vmax = _exact(q64, values, table, lengths, news, first, tokens)
    pos, seq = _positions(lengths, news)
    sees = (seq == 0) & (pos >= late * tokens)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    keep = np.ones(got.shape, dtype=bool)
    keep[sees, group:] = False
    _close(got, want, tol, vmax, dtype, keep)
    assert np.isnan(got[~keep]).all()
    assert np.isfinite(got_lse[:, ~sees]).all() and np.isfinite(got_lse[:group]).all()
    assert which == "v" or np.isnan(got_lse[group:][:, sees]).all()


@pytest.mark.parametrize("tokens", [16, 64])
@pytest.mark.parametrize("dtype,group,hd,news", FORMS)
def test_rows_in_front_of_a_spoilt_first_page_stay_empty(dtype, group, hd, news, tokens):
    """The first visible position is one of the new rows': the rows before it
    see nothing, also where its page is spoilt."""
    rng = np.random.default_rng(hd + tokens)
    first = [tokens * 9 + 5, 0]
    lengths = [first[0] + (news[0] + 1) // 2, news[1] + 133]
    lengths[0] = max(lengths[0], news[0])  # the new rows begin before it all the same
    assert lengths[0] - news[0] < first[0]
    cache, _, table = _filled(rng, lengths, 2, hd, tokens)
    _, q = _rows(rng, (sum(news), 2 * group, hd), dtype)
    for scale in (cache.k_scale, cache.v_scale):
        scale[int(table[0, first[0] // tokens])] = float("nan")
    out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), first=_i32(first),
                                   max_new=max(news), max_tokens=max(lengths))
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    pos, seq = _positions(lengths, news)
    blind, spoilt = (seq == 0) & (pos < first[0]), (seq == 0) & (pos >= first[0])
    assert blind.any() and not out[blind].any() and np.isneginf(lse[:, blind]).all()
    assert np.isnan(out[spoilt]).all() and np.isnan(lse[:, spoilt]).all() and np.isfinite(out[seq == 1]).all()


@pytest.mark.parametrize("k", [20, 28, 40, 100])
@pytest.mark.parametrize("tokens", [16, 32, 64])
@pytest.mark.parametrize("dtype,group,hd,news", FORMS)
def test_pages_that_a_row_does_not_see_do_not_move_its_precision(dtype, group, hd, news, tokens, k):
    """V scales 2^k larger behind a row's own position and in front of the
    first one seen: every row keeps the precision of what it sees."""
    rng = np.random.default_rng(hd + tokens + k)
    lengths = [news[0] + 75, news[1] + 133]
    first = [0, 100]
    cache, values, table = _filled(rng, lengths, 2, hd, tokens)
    q64, q = _rows(rng, (sum(news), 2 * group, hd), dtype)
    late, early = (lengths[0] - 2) // tokens, 100 // tokens - 1
    for page in (int(table[0, late]), int(table[1, early])):
        cache.v_scale[page, 1] *= 2.0 ** k
        values[1, page, 1] *= 2.0 ** k
    out, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), first=_i32(first),
                                 max_new=max(news), max_tokens=max(lengths))
    want, tol, vmax = _exact(q64, values, table, lengths, news, first, tokens)
    # what sees the large page may be past float16's numbers
    keep = np.broadcast_to(vmax < 6e4 if dtype == "float16" else vmax < np.inf, want.shape)
    _close(out.double().cpu().numpy(), want, tol, vmax, dtype, keep)


@pytest.mark.parametrize("max_tokens", [None, 100000])
@pytest.mark.parametrize("dtype,group,hd,news", FORMS)
def test_rows_that_no_sequence_owns_are_empty(dtype, group, hd, news, max_tokens):
    """A batch padded to a fixed number of rows, in front and behind; memory
    that held something else."""
    torch = _torch()
    rng = np.random.default_rng(hd)
    lengths = [n + 40 for n in news] + [17]
    cache, values, table = _filled(rng, lengths, 2, hd, 32)
    front, behind = 3, 7 + news[0]
    rows = front + sum(news) + behind
    q64, q = _rows(rng, (rows, 2 * group, hd), dtype)
    offsets = front + np.concatenate([_offsets(news), [sum(news)]])  # the last sequence brings nothing
    status = ops.new_status()
    for fill in (float("nan"), 7.0):
        dirty = [torch.full((rows * 2 * group * hd + i * 1000,), fill, device="cuda") for i in range(4)]
        del dirty
        out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(offsets), max_new=max(news),
                                       max_tokens=max_tokens, status=status)
        ops.check_status(status)
        owned = slice(front, front + sum(news))
        want, tol, vmax = _exact(q64[owned], values, table, lengths, news + [0], [0, 0, 0], 32)
        got = out.double().cpu().numpy()
        _close(got[owned], want, tol, vmax, dtype, np.ones(want.shape, dtype=bool))
        for outside in (slice(0, front), slice(front + sum(news), rows)):
            assert not got[outside].any() and torch.isneginf(lse[:, outside]).all()
    # numbers of the last sequence that do not fit: the rows behind it are not taken for results
    offsets[-1] -= 1
    out, lse = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(offsets), max_new=max(news),
                                   max_tokens=max_tokens, status=status)
    assert int(status.item()) == 8 and torch.isnan(out[front + sum(news):]).all()
    with pytest.raises(ops._lib.MeshError):
        ops.cache_attention(q, cache, _i32(table)[:0], _i32([]), _i32([0]))


def _workspace(batch, rows, q_heads, kv_heads, hd, max_new, max_tokens):
    import ctypes
    n = ctypes.c_size_t()
    ops.check(ops._lib.load().mb_op_cache_attention_workspace(batch, rows, q_heads, kv_heads, hd, 0, max_new, max_tokens,
                                                              ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("batch,rows,q_heads,kv_heads,hd,max_new", [(64, 4096 + 63 * 64, 64, 8, 128, 4096),
                                                                    (64, 64 * 2048, 8, 8, 128, 64 * 2048),
                                                                    (128, 131072, 8, 8, 96, 131072), (3, 700, 4, 2, 128, 700),
                                                                    (1, 100000, 8, 8, 128, 1)])
def test_workspace_follows_the_rows(batch, rows, q_heads, kv_heads, hd, max_new):
    """Not the batch times its longest prompt: FP32 sums of the rows there
    are, and a block a sequence."""
    assert _workspace(batch, rows, q_heads, kv_heads, hd, max_new, 4096) <= \
        2 * (rows * q_heads + batch * kv_heads * 256) * hd * 4 + 2e8


@pytest.mark.parametrize("hd,group,announced", [(128, 2, None), (96, 3, 700), (128, 1, 100000)])
def test_ragged_prompts_of_wide_single_precision(hd, group, announced):
    """One long prompt among short ones, nothing and single tokens: sums in
    the workspace that begin at any row, with the number of new rows given,
    not given and too large."""
    rng = np.random.default_rng(hd)
    news, tokens = [1, 700, 0, 129, 5, 260, 1, 511], 32
    lengths = [n + 41 * i for i, n in enumerate(news)]
    cache, values, table = _filled(rng, lengths, 2, hd, tokens)
    q64, q = _rows(rng, (sum(news), 2 * group, hd), "float32")
    out, _ = ops.cache_attention(q, cache, _i32(table), _i32(lengths), _i32(_offsets(news)), max_new=announced)
    want, tol, vmax = _exact(q64, values, table, lengths, news, [0] * len(news), tokens)
    _close(out.double().cpu().numpy(), want, tol, vmax, "float32", np.ones(want.shape, dtype=bool))


def test_rows_that_a_write_did_not_announce_are_reported():
    """max_new 0 with new rows: not a write of nothing with a clean status."""
    torch = _torch()
    cache = ops.new_kv_cache(2, 2, 32, 16)
    x = torch.ones((20, 2, 32), device="cuda")
    status = ops.new_status()
    ops.cache_write(cache, x, x, _i32([[0, 1]]), _i32([20]), _i32([0, 20]), max_new=0, status=status)
    assert int(status.item()) == 8
    # no new rows: nothing to report, however many rows stand behind
    status.zero_()
    ops.cache_write(cache, x, x, _i32([[0, 1]]), _i32([20]), _i32([0, 0]), max_new=0, status=status)
    assert int(status.item()) == 0


def test_empty_tensors_of_any_strides_are_taken():
    """Empty arrays of NumPy come with strides of 0: nothing to do, not an error."""
    torch = _torch()
    cache = ops.new_kv_cache(2, 3, 40, 16)
    rows = torch.from_numpy(np.random.default_rng(0).normal(0, 1, (0, 3, 40))).float().cuda()
    assert rows.stride(2) == 0
    status = ops.new_status()
    ops.cache_write(cache, rows, rows, _i32([[0, 1]]), _i32([20]), _i32([0, 0]), status=status)
    out, lse = ops.cache_attention(rows, cache, _i32([[0, 1]]), _i32([20]), _i32([0, 0]), status=status)
    assert out.shape == (0, 3, 40) and lse.shape == (3, 0)
    none = torch.from_numpy(np.random.default_rng(0).normal(0, 1, (0, 5))).cuda()
    r = ops.token_logprobs(none.float(), _i32([]), 2, status=status)
    assert r.top_index.shape == (0, 2)
    assert ops.token_logprobs_backward(none.float(), _i32([]), r.lse, r.entropy).shape == (0, 5)
    k, _ = ops.cache_read(cache, none.int(), _i32([]), 4, head_dim=40, status=status)
    assert k.shape == (0, 4, 3, 40)
    ops.check_status(status)
