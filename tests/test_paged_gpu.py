"""GPU: the paged cache's operators and beam search's selection (cudallm_b200/paged.py) against oracle/paged64.py.

Tolerances (eps = 2^-24, one rounding to fp32; errors of a sum of n terms taken as sqrt(n) eps times its size, with a
factor of 8 in hand):
  attention   a score is off by E = 8 eps sqrt(D) S, S = scale sum |q k|; so is ln of every weight, twice over with the sum:
              |out - ref| <= (2 E + 8 eps sqrt(T)) max|v|, |lse - ref| <= E + 8 eps sqrt(T) + 2 eps |lse|
  rotation    |y - ref| <= 8 eps factor (|a| + |b|)
  selection   |score - ref| <= 8 eps (|score| + |logit| + |lse| + sqrt(V))
each plus half a unit in the last place of the output's type (2^-11 fp16, 2^-8 bf16 relative, 2^-24 absolute), and integers
exactly."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from cudallm_b200 import paged
from cudallm_b200.abi import CudaLLMError
from oracle import paged64 as R

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HALF_ULP = {torch.float32: EPS, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _lib(native_lib):
    return native_lib


def _np(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _ints(a) -> torch.Tensor:
    return torch.from_numpy(np.array(a, np.int32)).cuda()


def _within(x: torch.Tensor, ref: np.ndarray, tol: np.ndarray) -> None:
    got = _np(x)
    assert got.shape == ref.shape
    assert np.array_equal(np.isfinite(got), np.isfinite(ref)) and np.array_equal(got[~np.isfinite(ref)], ref[~np.isfinite(ref)])
    with np.errstate(invalid="ignore"):
        off = np.abs(got - ref) - (tol + HALF_ULP[x.dtype] * np.abs(ref) + EPS)
    off = np.where(np.isfinite(ref), off, 0.0)
    assert off.max(initial=0.0) <= 0, f"over the tolerance by {off.max()}"


def _cache(layers, pages, kv_heads, page, dim, dtype, order="heads", fill=None, seed=0):
    shape = (layers, pages, kv_heads, page, dim) if order == "heads" else (layers, pages, page, kv_heads, dim)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(shape, generator=gen, device="cuda").to(dtype) if fill is None else torch.full(shape, fill, dtype=dtype, device="cuda")
            for _ in range(2))
    if order != "heads":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    return paged.PagedCache(k, v)


def _layout(lens, page, width=None, spare=2, seed=0):
    """A table with pages of its own for every row, anywhere in the pool."""
    counts = [-(-n // page) for n in lens]
    width = max(counts + [1]) if width is None else width
    pages = sum(counts) + spare
    ids, t, at = np.random.default_rng(seed).permutation(pages), np.full((len(lens), width), -1, np.int32), 0
    for r, n in enumerate(counts):
        t[r, :n] = ids[at:at + n]
        at += n
    return t, pages


def _poison(cache, table, lens, layer):
    """Fills every slot that no row uses with NaN and infinities, so that a read of one shows."""
    used = np.zeros((cache.n_pages, cache.page_size), bool)
    for r, n in enumerate(lens):
        for t in range(n):
            if 0 <= table[r][t // cache.page_size] < cache.n_pages:
                used[table[r][t // cache.page_size], t % cache.page_size] = True
    dirt = torch.from_numpy(~used).cuda()[None, :, None, :, None]
    cache.k.copy_(torch.where(dirt, float("nan"), cache.k))
    cache.v.copy_(torch.where(dirt, float("inf"), cache.v))


def _check_attend(cache, q, table, lens, *, layer=0, scale=None, window=0):
    out, lse = cache.attend(q, _ints(table), _ints(lens), layer=layer, scale=scale, window=window, with_lse=True)
    k = np.nan_to_num(_np(cache.k[layer]), nan=1e30, posinf=1e30)
    v = np.nan_to_num(_np(cache.v[layer]), nan=1e30, posinf=1e30)
    ref, ref_lse, size = R.attend64(_np(q), k, v, np.array(table), lens, scale, window)
    T = max(1, cache.page_size * np.array(table).shape[1])
    vmax = np.abs(np.where(v < 1e30, v, 0)).max()
    e = 8 * EPS * np.sqrt(cache.head_dim) * size
    _within(out, ref, ((2 * e + 8 * EPS * np.sqrt(T)) * vmax)[..., None])
    _within(lse, ref_lse, e + 8 * EPS * np.sqrt(T) + 2 * EPS * np.abs(np.where(np.isfinite(ref_lse), ref_lse, 0)))
    return out, lse


# ---- attention --------------------------------------------------------------------------------

@pytest.mark.parametrize("x, kv", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 64), (32, 4, 128), (8, 8, 64), (7, 1, 80), (16, 1, 64), (40, 1, 32), (6, 2, 256), (24, 2, 128), (3, 3, 8)])
@pytest.mark.parametrize("order, page", [("heads", 16), ("tokens", 24)])
def test_attend_types_and_heads(x, kv, heads, kv_heads, dim, order, page):
    lens = [0, 1, page - 1, page, page + 1, 130, 515]
    table, pages = _layout(lens, page)
    cache = _cache(2, pages, kv_heads, page, dim, kv, order, seed=heads)
    _poison(cache, table, lens, 1)
    q = torch.randn((len(lens), heads, dim), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(x)
    _check_attend(cache, q, table, lens, layer=1)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 31, 32, 33, 64, 128, 1000])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 100000])
def test_attend_page_sizes_and_windows(page, window):
    lens = [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 0, 1999]
    table, pages = _layout(lens, page)
    cache = _cache(1, pages, 2, page, 64, F16)
    _poison(cache, table, lens, 0)
    q = torch.randn((len(lens), 8, 64), device="cuda")
    _check_attend(cache, q, table, lens, window=window)


@pytest.mark.parametrize("lens", [[32768], [9000, 1, 20000, 0], [5] * 300, [700 + 3 * i for i in range(64)], [0, 0, 0]], ids=str)
def test_attend_lengths(lens):
    table, pages = _layout(lens, 64)
    cache = _cache(1, pages, 2, 64, 64, BF16)
    q = torch.randn((len(lens), 8, 64), device="cuda", dtype=BF16)
    a = _check_attend(cache, q, table, lens)
    b = cache.attend(q, _ints(table), _ints(lens), with_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # the same bits every time


def test_attend_missing_pages_are_masked():
    lens, page = [200, 200, 64, 500, 77], 16
    table, pages = _layout(lens, page)
    table[0, 3] = -1
    table[0, 0] = -7
    table[1, :] = -1  # nothing left
    table[2, :2] = [pages, 2 ** 31 - 1]
    table[3, 5:30] = -2 ** 31
    cache = _cache(1, pages, 2, page, 64, F16)
    _check_attend(cache, torch.randn((5, 8, 64), device="cuda"), table, lens)


def test_attend_clamps_lengths_to_the_table():
    table, pages = _layout([40, 40, 40], 8, width=5)
    cache = _cache(1, pages, 1, 8, 64, F16)
    q = torch.randn((3, 4, 64), device="cuda")
    _check_attend(cache, q, table, [10 ** 9, -5, -2 ** 31])


def test_attend_empty_table_and_no_rows():
    cache = _cache(1, 4, 1, 8, 64, F16)
    out, lse = cache.attend(torch.ones((2, 4, 64), device="cuda"), _ints(np.zeros((2, 0))), _ints([0, 3]), with_lse=True)
    assert torch.all(out == 0) and torch.all(torch.isneginf(lse))
    assert cache.attend(torch.ones((0, 4, 64), device="cuda"), _ints(np.zeros((0, 3))), _ints([])).shape == (0, 4, 64)


def test_attend_strided_and_broadcast_queries():
    lens = [70, 5, 33]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 2, 16, 64, F16)
    packed = torch.randn((3, 12, 64), device="cuda")
    _check_attend(cache, packed[:, 2:10], table, lens)
    _check_attend(cache, packed.view(-1)[5:5 + 3 * 700].view(3, 700)[:, 1:513].view(3, 8, 64), table, lens)  # rows of an odd stride, off alignment
    _check_attend(cache, packed[:1, :1].expand(3, 8, 64), table, lens)
    wide = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = _ints(table)
    a = cache.attend(packed[:, :8], wide[:, :table.shape[1]], _ints(lens))
    assert torch.equal(a, cache.attend(packed[:, :8].contiguous(), _ints(table), _ints(lens)))


def test_attend_more_rows_than_one_launch_takes():
    rng = np.random.default_rng(7)
    lens = [int(n) for n in rng.integers(0, 60, 2500)]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 1, 16, 64, F16)
    _check_attend(cache, torch.randn((2500, 4, 64), device="cuda"), table, lens)


def test_attend_peaked_and_tiny_scores():
    """One key far above the rest, at either end and inside; and scores of one size where the weights are all alike."""
    lens = [900] * 4
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 1, 16, 64, F16)
    k = cache.k[0, :, 0]
    for r, t in enumerate([0, 450, 899]):
        k[int(table[r][t // 16]), t % 16] = 6.0
    for p in table[3]:
        k[int(p)] = 0.0
    q = torch.full((4, 8, 64), 3.0, device="cuda")
    _check_attend(cache, q, table, lens)
    _check_attend(cache, 200 * q, table, lens)
    _check_attend(cache, q, table, lens, scale=0.0)
    _check_attend(cache, q, table, lens, scale=-0.05)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e6])
def test_attend_query_magnitudes(size):
    """fp32 queries far outside of the cache type's range; the scale brings the scores back."""
    lens = [333, 50]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 2, 16, 64, F16)
    q = size * torch.randn((2, 8, 64), device="cuda")
    q[:, ::2] *= 1e-3
    _check_attend(cache, q, table, lens, scale=0.125 / size)


def _tail_case(gap, rows, length, seed=0):
    """Rows over the same pages: a first token `gap` nats above all others with a value of 0, the others' values of one sign."""
    page, dim = 64, 64
    table, pages = _layout([length], page)
    cache = _cache(1, pages, 1, page, dim, F16, seed=seed)
    q = torch.randn(dim, generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
    cache.k.mul_(0.05)
    cache.v.abs_().add_(0.5)
    cache.k[0, int(table[0][0]), 0, 0] = q * (gap / (dim ** -0.5 * float(q @ q)))
    cache.v[0, int(table[0][0]), 0, 0] = 0.0
    return cache, q.expand(rows, 4, dim), np.repeat(table, rows, 0), [length] * rows


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("gap", [10, 12, 14, 16, 17, 18, 20])
@pytest.mark.parametrize("rows, length", [(1, 32768), (600, 8192)])
def test_attend_many_small_weights_over_fp16_pages(x, gap, rows, length):
    """The tail of a softmax under one large weight, in cut rows and in whole ones: what is left of the output is that tail, and has to keep its
    digits. A weight is off by 2 E (score, sum) and by the rounding of its two planes: 2^-22 of itself and, as the largest is 2^15 and fp16's
    grid 2^-24, 2^-40 of the largest; the lse as everywhere."""
    cache, q, table, lens = _tail_case(gap, rows, length)
    q = q.to(x)
    out, lse = cache.attend(q, _ints(table), _ints(lens), with_lse=True)
    ref, ref_lse, size = R.attend64(_np(q[:1]), _np(cache.k[0]), _np(cache.v[0]), table[:1], lens[:1])
    e = (8 * EPS * np.sqrt(cache.head_dim) * size)[..., None]
    tol = (2 * e + 8 * EPS * np.sqrt(length) + 2.0 ** -22) * np.abs(ref) + length * 2.0 ** -40 * np.abs(_np(cache.v)).max()
    many = lambda a: np.broadcast_to(a, (rows, *a.shape[1:]))  # noqa: E731
    _within(out, many(ref), many(tol))
    _within(lse, many(ref_lse), many(e[..., 0] + 8 * EPS * np.sqrt(length) + 2 * EPS * np.abs(ref_lse)))


@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("big, rest", [(64.0, 1.0), (4096.0, 1.0), (65536.0, 1.0), (3e38, 1e36), (1e-30, 1e-30)])
def test_attend_queries_with_one_large_dim(x, dim, big, rest):
    """One dim of the query far above the others where the keys are 0, so that the others alone make the scores: they are held to the same tolerance
    as without it. And queries at both ends of fp32's range."""
    lens = [700, 40]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 2, 16, dim, F16)
    cache.k[..., 3] = 0.0
    q = rest * torch.randn((2, 8, dim), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    q[..., 3] = big
    _check_attend(cache, q.to(x), table, lens, scale=dim ** -0.5 / rest)


@pytest.mark.parametrize("x, kv", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F16)])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 64), (8, 4, 128), (32, 2, 128), (6, 2, 256)])
def test_attend_queries_that_are_not_numbers(x, kv, heads, kv_heads, dim):
    """Their heads are not numbers either, out and lse alike, in rows that are cut and rows that are whole; every other head keeps its bits, and a row
    without a token is 0 and -inf as ever."""
    lens = [20000, 1, 700, 0, 64]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, kv_heads, 16, dim, kv)
    q = torch.randn((len(lens), heads, dim), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(x)
    bad = torch.zeros((len(lens), heads), dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 0] = bad[2, heads - 1] = bad[3, 2] = bad[4, 3] = bad[4, 4] = True
    dirty = q.clone()
    dirty[..., dim // 2] = torch.where(bad, float("nan"), q[..., dim // 2])
    ref, ref_lse = cache.attend(q, _ints(table), _ints(lens), with_lse=True)
    out, lse = cache.attend(dirty, _ints(table), _ints(lens), with_lse=True)
    bad[3] = False
    assert bool(torch.isnan(out[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    assert torch.equal(out[~bad], ref[~bad]) and torch.equal(lse[~bad], ref_lse[~bad])


def test_attend_offsets_past_32_bits():
    """Pages more than 2^32 elements into the pool."""
    page, dim, pages = 64, 128, 2 ** 32 // (64 * 128) + 300
    k = torch.empty((1, pages, 1, page, dim), dtype=F16, device="cuda")
    ids = [pages - 1, 3, pages - 200, 2 ** 31 // (64 * 128) + 1]
    k[0, ids] = torch.randn((4, 1, page, dim), device="cuda", dtype=F16)
    cache = paged.PagedCache(k, k)
    q = torch.randn((1, 4, dim), device="cuda")
    out = cache.attend(q, _ints([ids]), _ints([250]))
    small = k[:, ids].contiguous()
    ref = paged.PagedCache(small, small).attend(q, _ints([[0, 1, 2, 3]]), _ints([250]))
    assert torch.equal(out, ref)


def test_attend_on_a_stream_of_its_own_and_in_a_graph():
    lens = [3000, 10, 777]
    table, pages = _layout(lens, 16)
    cache = _cache(1, pages, 2, 16, 64, F16)
    q, t, n = torch.randn((3, 8, 64), device="cuda"), _ints(table), _ints(lens)
    ref = cache.attend(q, t, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [cache.attend(q, t, n) for _ in range(20)]
    here = [cache.attend(q, t, n) for _ in range(20)]  # both streams at once
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs + here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, t, n)
        out2 = cache.attend(q, t, n, window=100)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(out2, cache.attend(q, t, n, window=100))


# ---- rotary positions and the store to pages ----------------------------------------------------

def _check_append(cache, q, k, v, positions, table, rope, *, layer=0, rows=None, out=None):
    before_k, before_v = _np(cache.k).copy(), _np(cache.v).copy()
    q0, k0, v0 = (None if x is None else _np(x).copy() for x in (q, k, v))
    got = cache.append(q, k, v, _ints(positions), _ints(table), rope, layer=layer, rows=None if rows is None else _ints(rows), out=out)
    pos = np.array(positions, np.int64)
    inv = _np(rope.inv_freq) if rope else np.zeros(0)
    factor = rope.factor if rope else 1.0
    turn = lambda x: R.rotate64(x, pos, inv, rope is not None and rope.interleaved, factor)  # noqa: E731

    def tol(x):
        n = len(inv)
        t = np.zeros_like(x)
        i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rope is not None and rope.interleaved else (slice(0, n), slice(n, 2 * n))
        t[..., i] = t[..., j] = 8 * EPS * abs(factor) * (np.abs(x[..., i]) + np.abs(x[..., j]))
        return t

    if q is not None:
        _within(got, np.where((pos >= 0)[:, None, None], turn(q0), 0.0), tol(q0))
    k_tol, v_tol = np.zeros_like(before_k), np.zeros_like(before_v)
    rk, tk = turn(k0), tol(k0)
    for i, p in enumerate(pos):
        row = i if rows is None else rows[i]
        if p < 0 or not 0 <= row < len(table) or p // cache.page_size >= table.shape[1]:
            continue
        e = table[row][p // cache.page_size]
        if 0 <= e < cache.n_pages:
            before_k[layer, e, :, p % cache.page_size], k_tol[layer, e, :, p % cache.page_size] = rk[i], tk[i]
            before_v[layer, e, :, p % cache.page_size] = v0[i]
    if rope is None:
        before_k = _np(torch.from_numpy(before_k).to(cache.k.dtype))
    _within(cache.k, before_k, k_tol)
    np.testing.assert_array_equal(_np(cache.v), _np(torch.from_numpy(before_v).to(cache.v.dtype)))


@pytest.mark.parametrize("x, kv", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F16)])
@pytest.mark.parametrize("dim, rotary", [(64, 64), (128, 64), (80, 40), (64, 2), (256, 256), (8, 8), (48, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_append_layouts(x, kv, dim, rotary, interleaved, order):
    lens = [40, 33]
    table, pages = _layout([n + 5 for n in lens], 16)
    cache = _cache(2, pages, 2, 16, dim, kv, order)
    pos = [p for n in lens for p in range(n)]
    rows = [r for r, n in enumerate(lens) for _ in range(n)]
    qkv = torch.randn((len(pos), 7 + 2 + 2, dim), device="cuda").to(x)
    rope = paged.Rope.make(rotary, interleaved=interleaved, scaling="yarn", scale=8.0) if rotary else None
    _check_append(cache, qkv[:, :7], qkv[:, 7:9], qkv[:, 9:], pos, table, rope, layer=1, rows=rows)


@pytest.mark.parametrize("dim, offset, stride", [(64, 0, 64), (64, 1, 65), (64, 4, 68), (72, 2, 74), (64, 8, 72)])
def test_append_strides_and_in_place(dim, offset, stride):
    """Inputs off 16-byte alignment and with gaps between heads; q rotated in place and into a strided output."""
    n, heads = 19, 5
    table, pages = _layout([n], 8)
    cache = _cache(1, pages, 1, 8, dim, F16)

    def strided(h):
        return torch.randn(offset + n * h * stride, device="cuda", dtype=F16)[offset:].view(n, h, stride)[..., :dim]

    rope = paged.Rope.make(dim // 2 * 2)
    q, k, v = strided(heads), strided(1), strided(1)
    rows = [0] * n
    out = strided(heads)
    _check_append(cache, q, k, v, list(range(n)), table, rope, rows=rows, out=out)
    _check_append(cache, q, k, v, list(range(n)), table, rope, rows=rows, out=q)
    _check_append(cache, None, k, v, list(range(n)), table, rope, rows=rows)


@pytest.mark.parametrize("layout", ["token", "head", "each"])
def test_append_in_place_in_a_packed_projection(layout):
    """q, k and v of one buffer (heads side by side in a token, tokens in a head, or q, k and v of each head together), q turned in place."""
    n, heads = 21, 3
    table, pages = _layout([n], 8)
    cache = _cache(1, pages, heads, 8, 64, F16)
    if layout == "token":
        q, k, v = torch.randn((n, 3 * heads, 64), device="cuda", dtype=F16).split(heads, 1)
    elif layout == "head":
        q, k, v = torch.randn((3 * heads, n, 64), device="cuda", dtype=F16).transpose(0, 1).split(heads, 1)
    else:
        q, k, v = torch.randn((n, heads, 3 * 64), device="cuda", dtype=F16).split(64, 2)
    k0, v0 = k.clone(), v.clone()
    _check_append(cache, q, k, v, list(range(n)), table, paged.Rope.make(64), rows=[0] * n, out=q)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    for out in (k, v):
        with pytest.raises(CudaLLMError, match="overlap k or v"):
            cache.append(q.clone(), k, v, _ints(range(n)), _ints(table), None, rows=_ints([0] * n), out=out)


def test_append_output_between_the_queries():
    """A buffer whose tokens hold q, k, v and a place for the turned q: nothing of it overlaps."""
    n, heads = 21, 3
    table, pages = _layout([n], 8)
    cache = _cache(1, pages, heads, 8, 64, F16)
    q, k, v, out = torch.randn((n, 4 * heads, 64), device="cuda", dtype=F16).split(heads, 1)
    q0 = q.clone()
    _check_append(cache, q, k, v, list(range(n)), table, paged.Rope.make(64), rows=[0] * n, out=out)
    assert torch.equal(q, q0)


def test_append_one_token_a_row_padding_and_places_outside():
    table, pages = _layout([64] * 6, 16)
    table[2, 1] = -1
    table[3, 0] = pages
    cache = _cache(1, pages, 2, 16, 64, BF16)
    q, k, v = (torch.randn((6, h, 64), device="cuda") for h in (8, 2, 2))
    rope = paged.Rope.make(64)
    _check_append(cache, q, k, v, [0, -1, 17, 3, 64, 2 ** 31 - 1], table, rope)
    _check_append(cache, q, k, v, [5, -2 ** 31, 7, 8, 9, 10], table, rope, rows=[0, 1, -1, 6, 2 ** 31 - 1, 5])


@pytest.mark.parametrize("scaling", ["none", "linear", "llama3", "yarn"])
def test_append_long_positions(scaling):
    """Angles of a million radians, where the reduction to one turn decides; the angle itself is rounded to fp32 by definition."""
    pos = [0, 1, 104857, 105615, 105616, 131071, 999983, 2 ** 24 - 1]
    cache = _cache(1, 2, 1, 8, 64, F16)
    table = np.full((1, 2 ** 21), -1, np.int32)
    q, k, v = (torch.randn((8, h, 64), device="cuda") for h in (4, 1, 1))
    _check_append(cache, q, k, v, pos, table, paged.Rope.make(64, scaling=scaling, scale=32.0), rows=[0] * 8)


def test_append_many_tokens_and_none():
    lens = [1500, 1, 700]
    table, pages = _layout(lens, 24)
    cache = _cache(1, pages, 8, 24, 64, BF16)
    pos = [p for n in lens for p in range(n)]
    rows = [r for r, n in enumerate(lens) for _ in range(n)]
    q, k, v = (torch.randn((len(pos), h, 64), device="cuda", dtype=BF16) for h in (32, 8, 8))
    _check_append(cache, q, k, v, pos, table, paged.Rope.make(64), rows=rows)
    _check_append(cache, q[:0], k[:0], v[:0], [], table, paged.Rope.make(64))


def test_rope_matches_the_models_frequencies():
    from cudallm_b200.synth import llama3_inv_freq
    got = paged.Rope.make(64, scaling="llama3", scale=32.0).inv_freq.cpu().numpy()
    assert np.allclose(got, llama3_inv_freq(), rtol=4 * EPS, atol=0)


# ---- pages ------------------------------------------------------------------------------------

def _check_fork(cache, tables, lens, refs, parents, room, out=None):
    k0, v0 = _np(cache.k).copy(), _np(cache.v).copy()
    inputs = [_ints(x) for x in (tables, lens, refs, parents)]
    t, n, r, missing = cache.fork(*inputs, room=room, out=out)
    want_t, want_n, want_r, want_missing, copies = R.fork_ref(np.array(tables), lens, np.array(refs), parents, cache.page_size, room)
    for got, want in ((t, want_t), (n, want_n), (r, want_r), (missing, [want_missing])):
        np.testing.assert_array_equal(_np(got), np.array(want))
    for i, want in zip(inputs, (tables, lens, refs, parents)):
        np.testing.assert_array_equal(_np(i), np.array(want))
    for src, dst, tokens in copies:
        k0[:, dst, :, :tokens], v0[:, dst, :, :tokens] = k0[:, src, :, :tokens], v0[:, src, :, :tokens]
    np.testing.assert_array_equal(_np(cache.k), k0)
    np.testing.assert_array_equal(_np(cache.v), v0)
    return _np(t), _np(n), _np(r), int(missing)


@pytest.mark.parametrize("order, kv_heads, dim, page", [("heads", 8, 64, 16), ("tokens", 2, 80, 5), ("heads", 1, 8, 1), ("tokens", 3, 256, 64)])
def test_fork_walks_of_beams(order, kv_heads, dim, page):
    """A prompt becomes beams, which branch, die and grow; the references stay those of the tables."""
    rng = np.random.default_rng(page)
    cache = _cache(3, 300 if page > 1 else 2000, kv_heads, page, dim, F16, order)
    tables, lens, refs = (_np(x) for x in cache.rows(2, 40 if page > 1 else 200))
    parents = [0, 1]
    tables, lens, refs, missing = _check_fork(cache, tables, lens, refs, parents, 3 * page + 2)
    assert missing == 0
    lens = np.array([3 * page + 1, page], np.int32)
    parents = [0, 0, 0, 0, 1, 1, 1, 1]
    for step in range(12):
        room = int(rng.integers(0, 3)) + (2 * page if step == 5 else 0)
        tables, lens, refs, missing = _check_fork(cache, tables, lens, refs, parents, room)
        assert missing == 0
        held = tables[tables >= 0]
        np.testing.assert_array_equal(np.bincount(held, minlength=cache.n_pages), refs)
        lens = lens + min(room, 1)
        parents = np.concatenate([rng.integers(0, 4, 4), rng.integers(4, 8, 4)])
        if step % 4 == 3:
            parents[rng.integers(0, 8)] = -1  # one sequence ends
    tables, lens, refs, missing = _check_fork(cache, tables, lens, refs, [-1] * 3, 4)
    assert not refs.any() and not lens.any() and (tables == -1).all()


def test_fork_shared_tails_reserved_pages_and_references_of_others():
    cache = _cache(2, 32, 2, 4, 64, BF16)
    tables = [[3, 7, 9, 11, -1, -1], [3, 7, 9, -1, -1, -1], [20, -1, -1, -1, -1, -1], [-1, 5, 6, -1, 8, -1], [-1] * 6]
    refs = np.zeros(32, np.int32)
    for e in np.array(tables).ravel():
        if e >= 0:
            refs[e] += 1
    refs[8] = 0    # after a gap: not the row's
    refs[3] += 2   # held by someone else too
    refs[20] += 1
    lens = [9, 10, 4, 9, 0]
    for parents in ([0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [1, 1, 0], [3, 3, 3, 2, 2], [0, 0, 0, 5, -1, 99, 2 ** 31 - 1, -2 ** 31], []):
        for room in (0, 1, 3, 4, 9):
            _check_fork(cache, tables, lens, refs, parents, room)


def test_fork_when_pages_run_out_or_the_table_ends():
    cache = _cache(2, 6, 1, 4, 64, F16)
    tables, lens, refs = [[0, 1, 2], [3, 4, -1]], [10, 7], np.array([1, 1, 1, 1, 1, 0], np.int32)
    assert _check_fork(cache, tables, lens, refs, [0, 0, 0, 1, 1], 1)[3] == 2
    assert _check_fork(cache, tables, lens, refs, [0, 1], 1)[3] == 0
    assert _check_fork(cache, tables, lens, refs, [0, 1], 2 ** 31 - 1)[3] > 10 ** 8
    assert _check_fork(cache, tables, [10 ** 9, -3], refs, [0, 1, 1], 0)[3] == 0
    full = np.ones(6, np.int32)
    assert _check_fork(cache, tables, lens, full, [0, 0], 0)[3] == 1
    assert _check_fork(cache, tables, lens, refs, [-1, -1], 5)[3] == 0


def test_fork_many_rows_and_pages():
    rng = np.random.default_rng(5)
    rows, page, pages = 1500, 4, 9000
    lens = rng.integers(0, 20, rows)
    table, _ = _layout(list(lens), page, width=8)
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    cache = _cache(1, pages, 1, page, 8, F16)
    _check_fork(cache, table, lens, refs, rng.integers(-1, rows, 2500), 2)
    _check_fork(cache, table, lens, refs, rng.integers(0, 3, 30), 2)


def test_fork_into_the_other_half_of_a_pair():
    cache = _cache(1, 64, 2, 16, 64, F16)
    tables, lens, refs = cache.rows(4, 4)
    other = (*(torch.full_like(x, 77) for x in (tables, lens, refs)), torch.full((1,), 77, dtype=torch.int32, device="cuda"))
    state = cache.fork(tables, lens, refs, _ints([0, 1, 2, 3]), room=20, out=other)
    assert state is other and _np(state[2]).sum() == 8 and int(state[3]) == 0
    with pytest.raises(CudaLLMError, match="overlap"):
        cache.fork(*state[:3], _ints([0, 1, 2, 3]), out=state)


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("pages, share", [(1, 1.0), (7, 0.5), (500, 0.0), (500, 0.02), (500, 0.5), (500, 0.97), (500, 1.0), (3000, 0.3)])
def test_compact(pages, share, order):
    rng = np.random.default_rng(pages)
    cache = _cache(2, pages, 2, 4, 64, F16, order)
    used = np.nonzero(rng.random(pages) < share)[0]
    tables = rng.choice(np.concatenate([used, [-1, -5, pages, 2 ** 31 - 1]]), (5, 40)).astype(np.int32)
    refs = np.zeros(pages, np.int32)
    refs[used] = rng.integers(1, 5, len(used))
    k0, v0 = _np(cache.k).copy(), _np(cache.v).copy()
    t, r, live = cache.compact(_ints(tables), _ints(refs))
    want_t, want_r, want_live, moves = R.compact_ref(tables, refs)
    np.testing.assert_array_equal(_np(t), want_t)
    np.testing.assert_array_equal(_np(r), want_r)
    assert int(live) == want_live
    for src, dst in moves:
        k0[:, dst], v0[:, dst] = k0[:, src], v0[:, src]
    np.testing.assert_array_equal(_np(cache.k), k0)
    np.testing.assert_array_equal(_np(cache.v), v0)


@pytest.mark.parametrize("pages, layers, kv_heads", [(9000, 2, 2), (16384, 1, 1), (16385, 1, 1), (40000, 1, 1)])
def test_compact_large_pools(pages, layers, kv_heads):
    """Plans that do not fit one launch: many heads of pages to move, many pages."""
    rng = np.random.default_rng(pages)
    cache = _cache(layers, pages, kv_heads, 1, 8, F16)
    refs = (rng.random(pages) < 0.6).astype(np.int32) * rng.integers(1, 3, pages).astype(np.int32)
    tables = rng.integers(-1, pages, (3, 500)).astype(np.int32)
    k0, v0 = _np(cache.k).copy(), _np(cache.v).copy()
    t, r, live = cache.compact(_ints(tables), _ints(refs))
    want_t, want_r, want_live, moves = R.compact_ref(tables, refs)
    np.testing.assert_array_equal(_np(r), want_r)
    np.testing.assert_array_equal(_np(t), want_t)
    assert int(live) == want_live
    src, dst = (np.array(x) for x in zip(*moves))
    k0[:, dst], v0[:, dst] = k0[:, src], v0[:, src]
    np.testing.assert_array_equal(_np(cache.k), k0)
    np.testing.assert_array_equal(_np(cache.v), v0)


@pytest.mark.parametrize("pages, rows, n_out, layers, width", [(20000, 40, 60, 1, 12), (3000, 40, 60, 40, 12), (3000, 600, 700, 1, 12), (3000, 20, 20, 1, 1500)])
def test_fork_plans_that_do_not_fit_one_launch(pages, rows, n_out, layers, width):
    rng = np.random.default_rng(rows)
    page = 4
    lens = rng.integers(0, 30, rows)
    counts = [-(-int(n) // page) for n in lens]
    table, at = np.full((rows, width), -1, np.int32), 0
    ids = rng.permutation(pages)
    for r, n in enumerate(counts):
        table[r, :n] = ids[at:at + n]
        at += n
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    cache = _cache(layers, pages, 4, page, 8, F16)
    for room in (1, 9):
        _check_fork(cache, table, lens, refs, rng.integers(-1, rows, n_out), room)


def test_compact_keeps_attention():
    lens = [100, 37, 200]
    table, pages = _layout(lens, 16, spare=40)
    cache = _cache(1, pages, 2, 16, 64, F16)
    q = torch.randn((3, 8, 64), device="cuda")
    before = cache.attend(q, _ints(table), _ints(lens))
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    t, r, live = cache.compact(_ints(table), _ints(refs))
    assert int(t.max()) < int(live)
    assert torch.equal(cache.attend(q, t, _ints(lens)), before)


# ---- selection --------------------------------------------------------------------------------

def _check_beam(logits, scores, keep, finished=None, eos=0):
    got = paged.beam_select(logits, _f32(scores), keep=keep, finished=None if finished is None else _ints(finished), eos=eos)
    x = _np(logits)
    ref, parents, tokens = R.beam_ref(x, np.array(scores, np.float32).astype(np.float64), keep, finished, eos)
    np.testing.assert_array_equal(_np(got[1]), parents)
    np.testing.assert_array_equal(_np(got[2]), tokens)
    big = np.abs(x[np.isfinite(x)]).max(initial=0.0) + np.log(x.shape[1]) + np.sqrt(x.shape[1])
    _within(got[0], ref, 8 * EPS * (np.abs(np.where(np.isfinite(ref), ref, 0)) + 2 * big))


def _f32(a):
    return torch.from_numpy(np.array(a, np.float32)).cuda()


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("groups, beams, keep, vocab", [(1, 1, 1, 1), (1, 4, 8, 1000), (3, 5, 5, 32007), (2, 1, 64, 128256), (1, 64, 64, 4099), (2, 8, 16, 128256),
                                                        (4, 3, 7, 50), (1, 2, 6, 3), (1, 64, 64, 1), (5, 4, 1, 257)])
def test_beam_sizes(x, groups, beams, keep, vocab):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (3 * torch.randn((groups * beams, vocab), generator=gen, device="cuda")).to(x)
    scores = np.random.default_rng(vocab).normal(-5, 2, (groups, beams))
    _check_beam(logits, scores, keep)


def test_beam_many_groups():
    """More groups than the single launch has counters for."""
    logits = torch.randn((5000 * 2, 45), device="cuda", dtype=BF16)
    _check_beam(logits, np.random.default_rng(0).normal(-4, 1, (5000, 2)), 3)


@pytest.mark.parametrize("vocab", [5, 900, 70001])
def test_beam_ties_go_to_the_lower_row_then_token(vocab):
    keep = 9
    same = torch.zeros((4, vocab), device="cuda")
    _check_beam(same, [[0.0, 0.0, 0.0, 0.0]], keep)
    _check_beam(same, [[-1.0, 0.0, 0.0, -1.0]], keep)
    _check_beam(-same, [[-2.0, -2.0, -2.0, -2.0]], keep)
    few = torch.randint(0, 3, (4, vocab), device="cuda").to(BF16)
    few[1:] = few[0]
    few[2, ::2] *= -1.0  # zeros of both signs are equal
    few[2] = few[2].abs()
    _check_beam(few, [[-1.0, -1.0, -1.0, -1.0]], keep)


def test_beam_equal_zeros():
    x = torch.zeros((1, 300), device="cuda")
    x[0, ::3] = -0.0
    _check_beam(x, [[0.0]], 8)


def test_beam_rising_and_falling_rows():
    up = torch.arange(50000, device="cuda", dtype=torch.float32) / 5000
    _check_beam(torch.stack([up, up.flip(0)]), [[-1.0, -1.2]], 33)


def test_beam_masked_and_poisoned_rows():
    inf = float("inf")
    x = torch.randn((6, 5000), device="cuda")
    x[0] = -inf                     # nothing left
    x[1, 10:] = -inf                # fewer tokens than are kept
    x[2, 77] = float("nan")         # a row that is not a number
    x[3, 5] = inf
    x[4, :2500] = torch.finfo(F32).min
    scores = [[-1.0, -1.0, -1.0, -1.0, -1.0, -30.0]]
    _check_beam(x, scores, 20)
    _check_beam(x, [[-1.0, -1.0, -1.0, -1.0, -inf, float("nan")]], 20)
    _check_beam(x[:1], [[0.0]], 5)
    _check_beam(x[2:3], [[0.0]], 5)
    _check_beam(x[3:4], [[0.0]], 5)
    _check_beam(torch.full((2, 3000), -inf, device="cuda"), [[-inf, 0.0]], 4)


@pytest.mark.parametrize("x, ban", [(F32, -1e4), (F32, -1e9), (F32, -1e10), (F32, -1e30), (F32, -3.4028234663852886e38), (BF16, -1e30), (BF16, -3.3895313892515355e38),
                                    (F16, -65504.0)])
def test_beam_tokens_masked_by_large_numbers(x, ban):
    """Most tokens of a row masked by a number, so that whole parts of it hold nothing else: as if they were masked by -inf."""
    vocab, keep = 30011, 9
    logits = torch.randn((4, vocab), device="cuda").to(x)
    banned = torch.ones(vocab, dtype=torch.bool, device="cuda")
    banned[torch.arange(40, device="cuda") * 7 + 17000] = False
    scores = _f32([[-1.0, -2.0], [-3.0, -3.0]])
    got = paged.beam_select(logits.masked_fill(banned, ban), scores, keep=keep)
    ref = paged.beam_select(logits.masked_fill(banned, -float("inf")), scores, keep=keep)
    assert bool(torch.isfinite(got[0]).all()) and all(torch.equal(a, b) for a, b in zip(got, ref))
    _check_beam(logits.masked_fill(banned, -float("inf")), _np(scores), keep)
    _check_beam(torch.full((2, vocab), ban, dtype=x, device="cuda"), [[0.0, -1.0]], keep)  # every token


def test_beam_finished_rows():
    x = torch.randn((8, 3000), device="cuda")
    x[3] = float("nan")  # a finished beam's row is not read
    scores = np.random.default_rng(1).normal(-3, 1, (2, 4))
    _check_beam(x, scores, 8, finished=[[1, 0, 0, 1], [0, 0, 0, 0]], eos=2999)
    _check_beam(x, scores, 8, finished=[[1, 1, 1, 1], [1, 1, 0, 2]], eos=0)


def test_beam_strided_and_shared_rows():
    wide = torch.randn((8, 1101), device="cuda", dtype=BF16)
    _check_beam(wide[:, 1:1001], [[-1.0] * 4, [-2.0] * 4], 5)
    _check_beam(wide[::2, 3:1000], [[-1.0] * 4], 5)
    _check_beam(wide[:1].expand(4, 1101), [[-1.0, -1.5, -2.0, -2.5]], 8)


@pytest.mark.parametrize("groups, vocab", [(3, 5000), (20, 128256)])
def test_beam_scores_in_place(groups, vocab):
    """One launch and two: the new scores written over the old ones, as many of them."""
    x, s = torch.randn((groups * 4, vocab), device="cuda"), _f32(np.random.default_rng(6).normal(-5, 1, (groups, 4)))
    ref = paged.beam_select(x, s, keep=4)
    out = (s, *(torch.empty_like(ref[1]) for _ in range(2)))
    got = paged.beam_select(x, s, keep=4, out=out)
    assert got is out and all(torch.equal(a, b) for a, b in zip(got, ref))


def test_beam_same_bits_in_a_graph_and_on_two_streams():
    x, s = torch.randn((16, 128256), device="cuda"), _f32(np.random.default_rng(2).normal(-5, 1, (4, 4)))
    ref = paged.beam_select(x, s, keep=8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = [paged.beam_select(x, s, keep=8) for _ in range(10)]
    here = [paged.beam_select(x, s, keep=8) for _ in range(10)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.beam_select(x, s, keep=8)
    graph.replay()
    torch.cuda.synchronize()
    for got in there + here + [out]:
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_a_step_in_a_graph():
    """A whole step of beams (fork, append, attend, select) captured once and replayed on new inputs equals the same calls."""
    G, W, heads, vocab = 2, 3, 8, 5000
    rows = G * W
    cache, other = (_cache(2, 200, 2, 8, 64, F16, fill=0.0) for _ in range(2))
    rope = paged.Rope.make(64)
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    state = cache.fork(*cache.rows(rows, 20), _ints(range(rows)), room=11)
    state = (state[0], torch.full_like(state[1], 10), state[2])
    qkv, logits, scores, parents = rand(rows, heads + 4, 64), rand(rows, vocab), rand(G, W), _ints([0, 0, 1, 3, 5, 5])

    def step(c):
        t, n, r, missing = c.fork(*state, parents, room=1)
        outs = []
        for layer in range(2):
            q = c.append(qkv[:, :heads], qkv[:, heads:heads + 2], qkv[:, heads + 2:], n, t, rope, layer=layer)
            outs += [q, c.attend(q, t, n + 1, layer=layer)]
        return [t, n, r, missing, *outs, *paged.beam_select(logits, scores, keep=W), c.k, c.v]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache)
    for _ in range(3):
        for x in (qkv, logits, scores):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        parents.copy_(_ints([0, 2, 2, 4, 3, 3]))
        for c in (cache, other):
            c.k.zero_()
            c.v.zero_()
        graph.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_beam_workspaces_of_threads(monkeypatch):
    """Threads that call on one stream each bring a workspace of their own. Nothing is launched here: the calls only show what they would pass."""
    seen, both = [], threading.Barrier(2)
    select, size = paged._beam_calls()
    monkeypatch.setattr(paged, "_beam_calls", lambda: (lambda ref, stream: seen.append((ref._obj.workspace, stream)) or 0, size))
    x, s = torch.zeros((64, 128256), device="cuda"), torch.zeros((8, 8), device="cuda")

    def call():
        both.wait()
        paged.beam_select(x, s, keep=8)
        both.wait()  # neither is over before the other has called

    paged.beam_select(x, s, keep=8)  # this thread's
    threads = [threading.Thread(target=call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 3 and len({stream for _, stream in seen}) == 1 and len({workspace for workspace, _ in seen}) == 3


def test_beam_from_several_threads():
    """Four threads select from logits of their own on one stream, in the form of two launches; each gets what it gets alone."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    xs = [torch.randn((64, 128256), generator=gen, device="cuda") for _ in range(4)]
    s = torch.zeros((8, 8), device="cuda")
    refs = [paged.beam_select(x, s, keep=8) for x in xs]
    torch.cuda.synchronize()
    found = [[] for _ in xs]
    threads = [threading.Thread(target=lambda i=i: found[i].extend(paged.beam_select(xs[i], s, keep=8) for _ in range(100))) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for got, ref in zip(found, refs):
        assert len(got) == 100 and all(torch.equal(a, b) for g in got for a, b in zip(g, ref))


def test_the_documented_loop_over_beams():
    """The loop in the module's documentation, run as it stands for several steps: every row holds its ancestors' keys in order and sees all of them."""
    loop = "".join(line[4:] for line in paged.__doc__.splitlines(keepends=True) if line.startswith("    "))
    G, beams, steps, page, vocab = 2, 3, 11, 4, 500
    cache = _cache(1, 80, 2, page, 64, F16, fill=0.0)
    tables, lens, refs = cache.rows(G, 8)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    ns = dict(cache=cache, beam_select=paged.beam_select, layers=1, rope=None, beams=beams, tables=tables, lens=lens, refs=refs,
              parents=_ints([[0] * beams, [1] * beams]), scores=torch.zeros((G, beams), device="cuda"))
    texts = [[] for _ in range(G)]
    for step in range(steps):
        texts = [list(texts[p]) for p in ns["parents"].view(-1).tolist()]
        ns.update(q=rand(G * beams, 4, 64), k=rand(G * beams, 2, 64).half().float(), v=rand(G * beams, 2, 64).half().float(), logits=rand(G * beams, vocab))
        exec(compile(loop, "loop", "exec"), ns)
        assert int(ns["missing"]) == 0 and ns["lens"].tolist() == [step + 1] * (G * beams)
        for r, text in enumerate(texts):
            text.append((ns["k"][r], ns["v"][r]))
            k, v = (_np(torch.stack([t[i] for t in text], 1))[None] for i in range(2))  # one page of all tokens
            ref, _, size = R.attend64(_np(ns["q"][r:r + 1]), k, v, np.array([[0]]), [len(text)])
            _within(ns["out"][r:r + 1], ref, ((16 * EPS * np.sqrt(64) * size + 8 * EPS * np.sqrt(len(text))) * np.abs(v).max())[..., None])


# ---- refusals ---------------------------------------------------------------------------------

def test_numbers_beyond_32_bits_are_refused():
    """They must not come out as other, valid numbers in the C structs."""
    cache = _cache(2, 8, 2, 16, 64, F16)
    t, n, r = cache.rows(2, 3)
    q, k, pos = torch.zeros((2, 8, 64), device="cuda"), torch.zeros((2, 2, 64), device="cuda"), _ints([0, 0])
    big = 2 ** 32
    for call in (lambda: cache.attend(q, t, n, layer=big), lambda: cache.attend(q, t, n, window=big), lambda: cache.append(q, k, k, pos, t, None, layer=big + 1),
                 lambda: cache.fork(t, n, r, pos, room=big), lambda: paged.beam_select(q[0], _f32([[0.0] * 8]), keep=big + 1),
                 lambda: paged.beam_select(q[0], _f32([[0.0] * 8]), keep=1, finished=_ints([[0] * 8]), eos=big), lambda: cache.attend(q, t, n, scale=1e300)):
        with pytest.raises(CudaLLMError) as e:
            call()
        assert e.value.code == 1


def test_sizes_beyond_32_bits_are_refused():
    """Neither may a tensor's sizes come out as others: a row of 2^32 + 5 logits is not one of 5."""
    cache = _cache(2, 8, 2, 16, 64, F16)
    t, n, r = cache.rows(2, 3)
    q = torch.zeros((1, 1, 64), device="cuda")
    logits = torch.empty((1, 2 ** 32 + 5), dtype=F16, device="cuda")
    for call in (lambda: paged.beam_select(logits, _f32([[0.0]]), keep=2), lambda: cache.attend(q.expand(1, 2 ** 32 + 4, 64), t[:1], n[:1]),
                 lambda: cache.compact(t.new_empty((0, 2 ** 32 + 3)), r), lambda: cache.fork(t.new_empty((0, 2 ** 32 + 3)), n[:0], r, n[:0])):
        with pytest.raises(CudaLLMError) as e:
            call()
        assert e.value.code == 1


def test_refusals():
    cache = _cache(2, 8, 2, 16, 64, F16)
    t, n, r = cache.rows(2, 3)
    q, k = torch.zeros((2, 8, 64), device="cuda"), torch.zeros((2, 2, 64), device="cuda")
    rope = paged.Rope.make(64)
    pos = _ints([0, 0])
    bad = [
        lambda: cache.attend(q, t, n, layer=2),
        lambda: cache.attend(q, t, n, layer=-1),
        lambda: cache.attend(q[:, :5], t, n),                     # 5 heads for 2 key heads
        lambda: cache.attend(q[:, :, :32], t, n),
        lambda: cache.attend(q.double(), t, n),
        lambda: cache.attend(q.cpu(), t, n),
        lambda: cache.attend(q, t[:1], n),
        lambda: cache.attend(q, t.long(), n),
        lambda: cache.attend(q, t, n[:1]),
        lambda: cache.attend(q, t, n, window=-1),
        lambda: cache.attend(q, t, n, scale=float("nan")),
        lambda: cache.attend(q, t, n, out=q),
        lambda: cache.attend(q, t, n, out=q.half()),
        lambda: cache.attend(q.transpose(1, 2).contiguous().transpose(1, 2), t, n),
        lambda: cache.append(q, k[:1], k, pos, t, rope),
        lambda: cache.append(q, k, k.half(), pos, t, rope),
        lambda: cache.append(q, k[:, :1], k[:, :1], pos, t, rope),
        lambda: cache.append(q, k, k, pos.long(), t, rope),
        lambda: cache.append(q, k, k, pos, t, paged.Rope.make(128)),
        lambda: cache.append(q, k, k, pos, t, rope, layer=2),
        lambda: cache.append(q[:, :7], k, k, pos, t, rope, out=q[:, 1:]),  # neither q itself nor apart from it
        lambda: cache.append(q, k, k, pos, t, rope, out=q[:1, :1].expand(2, 8, 64)),
        lambda: cache.fork(t, n, r[:4], pos),
        lambda: cache.fork(t, n, r, pos, room=-1),
        lambda: cache.fork(t, n, r, pos.long()),
        lambda: cache.fork(t, n, r, pos, out=(t, n.clone(), r.clone(), pos[:1].clone())),
        lambda: cache.compact(t, r, out=(t.clone(), r, pos[:1].clone())),
        lambda: cache.compact(t, r.long()),
        lambda: paged.beam_select(q[0], _f32([[0.0] * 8]), keep=0),
        lambda: paged.beam_select(q[0], _f32([[0.0] * 8]), keep=65),
        lambda: paged.beam_select(q[0], _f32([[0.0] * 7]), keep=1),
        lambda: paged.beam_select(q[0, :, :1], _f32([[0.0] * 8]), keep=9),
        lambda: paged.beam_select(q[0], _f32([[0.0] * 8]), keep=1, finished=_ints([[0] * 8]), eos=64),
        lambda: paged.beam_select(q[0].double(), _f32([[0.0] * 8]), keep=1),
        lambda: paged.PagedCache(cache.k, cache.v[:, :, :, :8]),
        lambda: paged.PagedCache(cache.k.float(), cache.v.float()),
        lambda: paged.PagedCache(cache.k[..., :60], cache.v[..., :60]),
        lambda: paged.PagedCache(cache.k.transpose(3, 4), cache.v.transpose(3, 4)),
        lambda: paged.PagedCache(cache.k[:1].expand(2, -1, -1, -1, -1), cache.v[:1].expand(2, -1, -1, -1, -1)).attend(q, t, n),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(CudaLLMError) as e:
            call()
        assert e.value.code == 1, i
    torch.cuda.synchronize()
