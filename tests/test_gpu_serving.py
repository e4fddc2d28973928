"""Drafted decoding on the GPU against plain 64-bit forms: the quantised cache,
the shared-prefix attention, the verification of drafts, and the three together."""

import ctypes
import math

import numpy as np
import pytest

from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
PAGE = 64


@pytest.fixture(scope="module")
def nb(native_built):
    import rustyneedle_b200

    return rustyneedle_b200


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def int32(torch, x, device="cuda:0"):
    return torch.tensor(np.asarray(x, dtype=np.int64).astype(np.int32), device=device)


def dtype_of(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def paged(rng, lengths, before=0, spare=3):
    """(prefix pages, table, pages): shuffled page tables; unused entries name pages outside the pool."""
    need = [-(-t // PAGE) for t in lengths]
    total = before + sum(need) + spare
    order = rng.permutation(total).astype(np.int32)
    table = np.full((len(lengths), max(1, max(need, default=1))), -1, dtype=np.int32)
    at = before
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    return order[:before].copy(), table, total


def make_batch(nb, torch, rows, lengths, table, /, **more):
    more = {"rows": int(sum(rows)), "max_rows": int(max(rows, default=0)), "max_length": int(max(lengths, default=0)), **more}
    return nb.KvBatch(int32(torch, starts(rows)), int32(torch, lengths), int32(torch, table), **more)


def random_rows(rng, torch, rows, heads, dim, dtype, strided=False):
    x = rng.standard_normal((rows, heads, dim)) * np.exp(rng.standard_normal((rows, heads, 1))) * np.exp(0.5 * rng.standard_normal((1, heads, dim)))
    t = torch.tensor(x, dtype=torch.float32, device="cuda:0").to(dtype)
    if strided:  # odd distances: no wide access is possible
        room = torch.full((rows, heads, dim + 5), float("nan"), dtype=dtype, device="cuda:0")
        room[:, :, 3 : 3 + dim] = t
        t = room[:, :, 3 : 3 + dim]
    return t


def numbers(t):
    return t.detach().to("cpu").double().numpy()


# ------------------------------------------------------------------------------------------------ cache: append, read

CACHE_CASES = [  # rows of each sequence, positions before them
    ([1], [0]), ([1], [63]), ([1], [64]), ([3, 0, 5, 1], [0, 10, 62, 200]), ([130], [0]), ([65, 1, 17], [63, 64, 31]), ([0, 0], [5, 0]),
    ([2] * 70, list(range(70))), ([5, 16, 33, 48], [3, 16, 15, 1]),
    # many rows: blocks of 16 rows with every alignment of their positions, across pages and sequences
    ([2000 + i for i in range(6)], [0, 1, 2, 3, 17, 50]), ([7, 900, 0, 1, 4000, 33, 3500, 16], [5, 62, 3, 0, 6, 127, 1, 48]),
]


def held(x, kind, dtype, torch):
    codes, scale = ref.quantise(x, kind)
    # the product of a code and an f32 scale is rounded to f32, then to the type: code and scale make it exact to 32
    # bits (int8: 7 + 24 bits, one rounding) and a type of fewer bits rounds that value
    y = (codes * scale[..., None]).astype(np.float32)
    return numbers(torch.tensor(y).to(dtype))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(CACHE_CASES)))
def test_rows_are_held_exactly(nb, torch, kind, dtype, case):
    rows, past = CACHE_CASES[case]
    rng = np.random.default_rng(100 + case)
    dim, kv = (64, 3) if case % 2 else (128, 2)
    lengths = [r + p for r, p in zip(rows, past)]
    _, table, pages = paged(rng, lengths)
    t = dtype_of(torch, dtype)
    n = sum(rows)
    keys = random_rows(rng, torch, n + 2, kv, dim, t, strided=case % 3 == 1)
    values = random_rows(rng, torch, n + 2, kv, dim, t)
    with nb.KvCache(kv, dim, pages, format=kind, device=0) as cache:
        batch = make_batch(nb, torch, rows, lengths, table)
        cache.append(batch, keys, values)
        out = [torch.full((n + 2, kv, dim), 7.0, dtype=t, device="cuda:0") for _ in range(2)]
        cache.read(batch, *out)
        cache.check()
        for x, y in zip((keys, values), out):
            assert np.array_equal(numbers(y[:n]), held(numbers(x[:n]), kind, t, torch))
            assert bool((y[n:] == 7.0).all())  # rows behind the last sequence stay
        # all positions at once: earlier ones are untouched rows of zeros
        whole = make_batch(nb, torch, lengths, lengths, table)
        back = [torch.empty(sum(lengths), kv, dim, dtype=torch.float32, device="cuda:0") for _ in range(2)]
        cache.read(whole, *back)
        at = 0
        for b, (r, p) in enumerate(zip(rows, past)):
            for x, y in zip((keys, values), back):
                assert not bool(y[at : at + p].any())
                got = numbers(y[at + p : at + p + r])
                assert np.array_equal(got, held(numbers(x[starts(rows)[b] : starts(rows)[b] + r]), kind, torch.float32, torch))
            at += r + p


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_special_rows(nb, torch, kind):
    dim, kv = 64, 1
    rng = np.random.default_rng(3)
    x = rng.standard_normal((16, kv, dim)).astype(np.float32)
    x[0] = 0
    x[1, 0, 5] = np.nan
    x[2, 0, 63] = np.inf
    x[3, 0, 0] = -np.inf
    x[4] *= 2.0**41
    x[5] *= np.float32(2.0**-70)
    x[6] = np.float32(2.0**-149)
    x[7, 0] = np.arange(64) - 32 + 0.5  # halves of the scale
    x[7, 0, 0] = 127
    x[8, 0] = (np.arange(64) % 32 - 16) * np.float32(0.03125)
    x[9] = np.float32(448) * np.float32(2.0**-3)
    x[10] = np.nextafter(np.float32(448), np.float32(500))
    x[11, 0] = np.float32(3.4e38)
    x[12] = -0.0
    # quotients next to a half: x = fl((k + 1/2) * scale) and its neighbours
    scale = np.float32(1.7) * (np.float32(1) / np.float32(127))
    k = np.arange(60).astype(np.float64) + 0.5
    for row, shift in ((13, -1), (14, 0), (15, 1)):
        y = (k * np.float64(scale)).astype(np.float32)
        if shift:
            y = np.nextafter(y, np.float32(shift * 1e9))
        x[row, 0, :60] = y
        x[row, 0, 60:] = np.float32(1.7)
    cache = nb.KvCache(kv, dim, 2, format=kind, device=0)
    batch = make_batch(nb, torch, [16], [16], np.array([[1]]))
    keys = torch.tensor(x, device="cuda:0")
    cache.append(batch, keys, keys.flip(0).contiguous())
    out = [torch.empty(16, kv, dim, device="cuda:0") for _ in range(2)]
    cache.read(batch, *out)
    want = held(x, kind, torch.float32, torch)
    assert np.array_equal(numbers(out[0]), want, equal_nan=True)
    assert np.array_equal(numbers(out[1]), want[::-1], equal_nan=True)
    assert np.isnan(want[[1, 2, 3, 4, 11]]).all() and np.isfinite(np.delete(want, [1, 2, 3, 4, 11], 0)).all()
    cache.check()


def test_a_page_far_into_a_large_pool(nb, torch):
    """Byte offsets past 32 bits (8 heads of 128: 64 KiB of key codes a page)."""
    pages = 70001
    cache = nb.KvCache(8, 128, pages, device=0)
    rng = np.random.default_rng(4)
    table = np.array([[pages - 1, 3, 65536]])
    keys, values = (random_rows(rng, torch, 150, 8, 128, torch.bfloat16) for _ in range(2))
    batch = make_batch(nb, torch, [150], [150], table)
    cache.append(batch, keys, values)
    out = [torch.empty_like(keys) for _ in range(2)]
    cache.read(batch, *out)
    for x, y in zip((keys, values), out):
        assert np.array_equal(numbers(y), held(numbers(x), "int8", torch.bfloat16, torch))
    query = random_rows(rng, torch, 150, 16, 128, torch.bfloat16)
    check_attend(nb, torch, cache, query, keys, values, [150], [150], table)
    cache.check()
    cache.close()


def test_bad_pages_and_sequences_are_left_out_and_reported(nb, torch):
    rng = np.random.default_rng(8)
    kv, dim = 2, 64
    cache = nb.KvCache(kv, dim, 6, device=0)
    rows, lengths = [3, 4, 70], [10, 70, 70]
    table = np.array([[0, -1], [1, 99], [2, 6]])  # the 2nd sequence's rows straddle into page 99, the 3rd's into 6
    keys, values = (random_rows(rng, torch, 77, kv, dim, torch.float32) for _ in range(2))
    batch = make_batch(nb, torch, rows, lengths, table)
    cache.append(batch, keys, values)
    with pytest.raises(nb.NeedleError) as e:
        cache.check()
    assert e.value.status == -4 and "page" in e.value.message
    cache.check()  # cleared
    out = [torch.full((77, kv, dim), 9.0, device="cuda:0") for _ in range(2)]
    cache.read(batch, *out)
    with pytest.raises(nb.NeedleError):
        cache.check()
    want = held(numbers(keys), "int8", torch.float32, torch)
    got = numbers(out[0])
    assert np.array_equal(got[:3], want[:3]) and np.array_equal(got[7 : 7 + 64], want[7 : 7 + 64])
    assert (got[3:7] == 9).all() and (got[71:] == 9).all()
    # masked pages: a sequence all of whose pages are bad has nothing to attend to
    query = random_rows(rng, torch, 77, 4, dim, torch.bfloat16)
    result = torch.full((77, 4, dim), 5.0, dtype=torch.bfloat16, device="cuda:0")
    bad = make_batch(nb, torch, rows, lengths, np.array([[0, -1], [77, 99], [2, 6]]))
    cache.attend(bad, query, result)
    with pytest.raises(nb.NeedleError):
        cache.check()
    assert not bool(result[3:7].any()) and bool(torch.isfinite(result).all())
    # a sequence out of its bounds: the others are served
    for rows2, lengths2, more in (([3, 4, 2], [10, 3, 20], {}), ([3, 9, 2], [10, 20, 20], {"max_rows": 5}), ([3, 4, 2], [10, 500, 20], {"max_length": 60}),
                                  ([3, 4, 2], [10, 200, 20], {"max_length": 300})):
        n = sum(rows2)
        mixed = make_batch(nb, torch, rows2, lengths2, np.array([[0, 1], [2, 3], [4, 5]]), **more)
        result.fill_(5.0)
        cache.append(mixed, keys, values)
        cache.attend(mixed, query, result)
        with pytest.raises(nb.NeedleError) as e:
            cache.check()
        assert "sequence" in e.value.message
        own = slice(rows2[0], rows2[0] + rows2[1])
        assert bool((result[own] == 5.0).all()) and bool((result[n:] == 5.0).all())
        assert not bool((result[: rows2[0]] == 5.0).all()) and not bool((result[n - 1] == 5.0).all())
    cache.close()


# -------------------------------------------------------------------------------------------------------------- attend


def check_attend(nb, torch, cache, query, keys, values, rows, lengths, table, prefix=0, prefix_pages=None, scale=None, out=None, bounds=None):
    """Attends and compares. keys and values hold the prefix's rows, then all positions of each sequence. `bounds` are the
    batch's, above its own.

    The bound for one element, to first order:
      half a step of the output's type, relative: eps / 2
      the f16 rounding of each weight w: 2^-11 of sum p |v|; a weight below f16's normal numbers is off by 2^-25 at most, with
        the largest weight (p vs, scaled) at 2^8 or above: 2^-33 of the largest p vs, times the code, summed over the keys
      a score's f32 products and sums: dim + 8 roundings (2^-23 each) of sum |q k| scale, and exp2's and log2's own error, 2^-20;
        a weight's error enters the sum above and the one below it
      the f32 sums over the keys: 2^-23 for each of n / 8 products and 16 joins."""
    t = query.dtype
    scale_ = 1 / math.sqrt(query.shape[2]) if scale is None else scale
    n = sum(rows)
    result = torch.full_like(query, 3.0) if out is None else out
    batch = make_batch(nb, torch, rows, lengths, table, **(bounds or {}))
    cache.attend(batch, query, result, prefix_pages, prefix, scale)
    cache.check()
    kc, ks = ref.quantise(numbers(keys), cache.format)
    vc, vs = ref.quantise(numbers(values), cache.format)
    want, mass, size, least = ref.attend(numbers(query[:n]), kc * ks[..., None], vc, vs, rows, lengths, prefix, scale_)
    most = prefix + max(lengths, default=0)
    score = 2 * ((query.shape[2] + 8) * 2.0**-23 * size + 2.0**-20)
    bound = torch.finfo(t).eps / 2 * np.abs(want) + mass * (2.0**-11 + score + (most / 8 + 16) * 2.0**-23) + 2.0**-33 * least + float(torch.finfo(t).smallest_normal) * 2.0**-8
    got = numbers(result[:n])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off, bound = np.where(np.isnan(want), 0, np.abs(got - want)), np.where(np.isnan(want), 0, bound)  # NaN is compared above
    worst = np.unravel_index(np.argmax(off - bound), off.shape) if off.size else None
    assert off.size == 0 or off[worst] <= bound[worst], (worst, off[worst], bound[worst], want[worst])
    assert bool((result[n:] == 3.0).all())
    return result


def attend_case(nb, torch, seed, rows, lengths, prefix, heads, kv, dim, kind, dtype, strided=False, scale=None, change=None, bounds=None):
    rng = np.random.default_rng(seed)
    t = dtype_of(torch, dtype)
    prefix_pages, table, pages = paged(rng, lengths, -(-prefix // PAGE))
    keys = random_rows(rng, torch, prefix + sum(lengths), kv, dim, t)
    values = random_rows(rng, torch, prefix + sum(lengths), kv, dim, t)
    query = random_rows(rng, torch, (bounds or {}).get("rows", sum(rows) + 1), heads, dim, t, strided)
    if change:
        change(query, keys, values)
    cache = nb.KvCache(kv, dim, pages, format=kind, device=0)
    shared = int32(torch, prefix_pages)
    if prefix:
        cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), keys[:prefix], values[:prefix])
    if sum(lengths):
        cache.append(make_batch(nb, torch, lengths, lengths, table), keys[prefix:], values[prefix:])
    out = torch.full_like(query, 3.0)
    if strided:
        out = torch.full((heads, query.shape[0], dim + 2), 3.0, dtype=t, device="cuda:0")[:, :, :dim].transpose(0, 1)
    return check_attend(nb, torch, cache, query, keys, values, rows, lengths, table, prefix, shared, scale, out, bounds)


ATTEND_CASES = [  # rows, lengths, prefix, heads, kv heads
    ([1], [1], 0, 1, 1), ([1], [1], 1, 2, 1), ([1], [64], 64, 4, 4), ([1], [65], 63, 8, 4), ([1, 1, 1], [1, 33, 130], 200, 8, 2),
    ([5, 0, 1, 3], [5, 40, 64, 129], 77, 6, 2), ([17], [17], 0, 4, 2), ([40, 1], [100, 1], 31, 5, 1), ([1] * 40, list(range(1, 41)), 515, 8, 4),
    ([2] * 9, [700 + 13 * i for i in range(9)], 0, 3, 3), ([3, 2], [3, 2], 1000, 16, 2), ([1, 2], [2, 2], 4, 64, 1),
    ([70, 129, 0, 33], [70, 200, 5, 90], 150, 4, 2), ([150], [300], 300, 8, 1), ([1] * 150, [1 + i % 7 for i in range(150)], 260, 4, 2),
]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(ATTEND_CASES)))
def test_attend(nb, torch, kind, dtype, dim, case):
    rows, lengths, prefix, heads, kv = ATTEND_CASES[case]
    attend_case(nb, torch, 200 + case, rows, lengths, prefix, heads, kv, dim, kind, dtype, strided=case % 4 == 1)


# The kernel, its tiles and its split follow the batch's bounds: with these the tiles of 128 rows are taken for sequences
# and prefixes of any length, one tile or two to a block.
WIDE_BOUNDS = [{"rows": 8192, "max_rows": 2048, "max_length": 1 << 14}, {"rows": 4000, "max_rows": 150, "max_length": 1 << 17}]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(ATTEND_CASES)))
def test_attend_with_wide_bounds(nb, torch, kind, dtype, dim, case):
    rows, lengths, prefix, heads, kv = ATTEND_CASES[case]
    attend_case(nb, torch, 250 + case, rows, lengths, prefix, heads, kv, dim, kind, dtype, strided=case % 4 == 2, bounds=WIDE_BOUNDS[case % 2])


@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 255, 256, 257, 383, 640, 1025])
@pytest.mark.parametrize("tail", [1, 127, 128, 129, 257, 400])
def test_attend_at_the_edges_of_wide_tiles(nb, torch, prefix, tail):
    n, odd = prefix + tail, prefix % 2
    attend_case(nb, torch, n, [min(tail, 130), 1, min(tail, 64)], [tail, 1, tail], prefix, 4, 2, 64 if odd else 128, "int8" if tail % 2 else "e4m3", "fp16", bounds=WIDE_BOUNDS[n % 2])


@pytest.mark.parametrize("prefix", [127, 128, 129, 255, 256, 257, 383, 1025])
@pytest.mark.parametrize("batch", [3, 40, 64, 65, 130])
def test_attend_at_the_edges_of_tiles(nb, torch, prefix, batch):
    rng = np.random.default_rng(prefix + batch)
    attend_case(nb, torch, prefix * batch, [1] * batch, list(rng.integers(1, 80, batch)), prefix, 4, 2, 64 if batch % 2 else 128, "int8" if prefix % 2 else "e4m3", "bf16")


@pytest.mark.parametrize("rows", [15, 16, 31, 63, 64, 65, 127, 128, 200])
@pytest.mark.parametrize("before", [0, 1, 64, 190])
def test_attend_many_rows_of_one_sequence(nb, torch, rows, before):
    attend_case(nb, torch, rows * 7 + before, [rows, 2], [rows + before, 3], before, 4, 2, 128 if rows % 2 else 64, "int8", "fp16")


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 3.0])
def test_attend_scales(nb, torch, scale):
    attend_case(nb, torch, 40, [1, 4], [30, 60], 140, 4, 2, 64, "int8", "bf16", scale=scale)


def test_attend_rows_of_very_different_size(nb, torch):
    """Values of sizes 2^-30 to 2^30, also where the small ones have the weight; keys that make the scores large."""

    def change(query, keys, values):
        n = values.shape[0]
        values *= torch.exp2(torch.linspace(-30, 30, n, device="cuda:0"))[torch.randperm(n, device="cuda:0", generator=torch.Generator("cuda").manual_seed(1))][:, None, None].to(values.dtype)
        keys[n // 2] *= 8
        values[n // 3] = 0

    attend_case(nb, torch, 41, [1, 3], [50, 90], 333, 4, 2, 64, "int8", "bf16", change=change)
    attend_case(nb, torch, 42, [1, 3], [50, 90], 333, 4, 2, 128, "e4m3", "bf16", change=change)


def test_attend_a_row_that_could_not_be_held(nb, torch):
    """A NaN key row makes every row that sees it NaN, and no other; the prefix and the other sequence stay clean."""

    def change(query, keys, values):
        keys[100 + 20, 0, 3] = float("nan")  # position 20 of the first tail, kv head 0
        values[100 + 25, 1, 3] = float("inf")  # position 25, kv head 1

    out = numbers(attend_case(nb, torch, 43, [30, 30], [30, 30], 100, 4, 2, 64, "int8", "bf16", change=change)[:60])
    assert np.isnan(out[20:30, :2]).all() and np.isfinite(out[:20, :2]).all()
    assert np.isnan(out[25:30, 2:]).all() and np.isfinite(out[:25, 2:]).all() and np.isfinite(out[30:]).all()


@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attend_does_not_look_behind_the_end(nb, torch, rows, kind):
    """Positions behind a length and behind the prefix, and unseen later rows, hold rows that are NaN."""
    rng = np.random.default_rng(44)
    kv, dim, prefix, length = 2, 64, 70, rows + 9
    prefix_pages, table, pages = paged(rng, [length + 150], -(-(prefix + 100) // PAGE))
    cache = nb.KvCache(kv, dim, pages, format=kind, device=0)
    poison = torch.full((length + 400, kv, dim), float("nan"), dtype=torch.bfloat16, device="cuda:0")
    cache.append(make_batch(nb, torch, [prefix + 50], [prefix + 50], prefix_pages[None]), poison, poison)
    cache.append(make_batch(nb, torch, [length + 150], [length + 150], table), poison, poison)
    keys, values = (random_rows(rng, torch, prefix + length, kv, dim, torch.bfloat16) for _ in range(2))
    cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), keys[:prefix], values[:prefix])
    cache.append(make_batch(nb, torch, [length], [length], table), keys[prefix:], values[prefix:])
    query = random_rows(rng, torch, rows, 4, dim, torch.bfloat16)
    check_attend(nb, torch, cache, query, keys, values, [rows], [length], table, prefix, int32(torch, prefix_pages))


def test_attend_long_tails_and_a_long_prefix(nb, torch):
    attend_case(nb, torch, 45, [1, 2], [20000, 5000], 0, 4, 1, 64, "int8", "bf16")
    attend_case(nb, torch, 46, [1, 1], [1, 70], 30000, 4, 1, 128, "e4m3", "fp16")


def test_attend_many_keys_and_many_rows(nb, torch):
    """The largest tiles over more than one round of key tiles; parts joined in several shares."""
    attend_case(nb, torch, 52, [600, 1], [5000, 77], 0, 4, 2, 128, "int8", "bf16")
    attend_case(nb, torch, 53, [1] * 300, [3] * 300, 5000, 8, 2, 64, "e4m3", "fp16")
    attend_case(nb, torch, 54, [1], [70], 60000, 4, 1, 64, "int8", "bf16")
    attend_case(nb, torch, 55, [2] * 5, [9000 + 64 * i for i in range(5)], 0, 2, 2, 64, "int8", "fp16")


def test_attend_a_row_that_could_not_be_held_with_wide_bounds(nb, torch):
    def change(query, keys, values):
        keys[100 + 20, 0, 3] = float("nan")
        values[100 + 25, 1, 3] = float("inf")

    for bounds in WIDE_BOUNDS:
        out = numbers(attend_case(nb, torch, 56, [30, 30], [30, 30], 100, 4, 2, 128, "int8", "bf16", change=change, bounds=bounds)[:60])
        assert np.isnan(out[20:30, :2]).all() and np.isfinite(out[:20, :2]).all()
        assert np.isnan(out[25:30, 2:]).all() and np.isfinite(out[:25, 2:]).all() and np.isfinite(out[30:]).all()


def test_attend_with_wide_bounds_does_not_look_behind_the_end(nb, torch):
    rng = np.random.default_rng(57)
    kv, dim, prefix, rows = 2, 128, 70, 40
    length = rows + 9
    prefix_pages, table, pages = paged(rng, [length + 150], -(-(prefix + 100) // PAGE))
    cache = nb.KvCache(kv, dim, pages, format="e4m3", device=0)
    poison = torch.full((length + 400, kv, dim), float("nan"), dtype=torch.bfloat16, device="cuda:0")
    cache.append(make_batch(nb, torch, [prefix + 50], [prefix + 50], prefix_pages[None]), poison, poison)
    cache.append(make_batch(nb, torch, [length + 150], [length + 150], table), poison, poison)
    keys, values = (random_rows(rng, torch, prefix + length, kv, dim, torch.bfloat16) for _ in range(2))
    cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), keys[:prefix], values[:prefix])
    cache.append(make_batch(nb, torch, [length], [length], table), keys[prefix:], values[prefix:])
    for bounds in WIDE_BOUNDS:
        query = random_rows(rng, torch, bounds["rows"], 4, dim, torch.bfloat16)
        check_attend(nb, torch, cache, query, keys, values, [rows], [length], table, prefix, int32(torch, prefix_pages), bounds=bounds)


def test_attend_with_wide_bounds_leaves_out_bad_pages_and_sequences(nb, torch):
    """A page outside the pool counts as no keys, in the prefix and in a tail; a sequence out of its bounds gets nothing."""
    rng = np.random.default_rng(58)
    kv, dim = 2, 128
    cache = nb.KvCache(kv, dim, 8, device=0)
    keys, values = (random_rows(rng, torch, 128, kv, dim, torch.bfloat16) for _ in range(2))
    cache.append(make_batch(nb, torch, [128], [128], np.array([[0, 1]])), keys, values)
    for bounds in WIDE_BOUNDS:
        query = random_rows(rng, torch, bounds["rows"], 4, dim, torch.bfloat16)
        whole, part = (torch.full_like(query, 5.0) for _ in range(2))
        for result, table, prefix_pages in ((whole, [[0]], [1]), (part, [[0, 1000]], [1, -1])):
            batch = make_batch(nb, torch, [40], [64], np.array(table), **bounds)
            cache.attend(batch, query, result, int32(torch, prefix_pages), 64)
        cache.check()
        assert torch.equal(whole, part)
        batch = make_batch(nb, torch, [40], [100], np.array([[0, 1000]]), **bounds)  # rows 60 .. 99 of the 100 positions
        cache.attend(batch, query, part, int32(torch, [1, -1]), 128)
        with pytest.raises(nb.NeedleError):
            cache.check()
        cache.attend(make_batch(nb, torch, [40], [64], np.array([[0]]), **bounds), query, whole, int32(torch, [1]), 64)
        cache.check()
        # rows 60 .. 99 see all of the 64 positions whose page is there, and so does row 63 of the other batch. The prefixes'
        # lengths split the keys differently, so both are off from the same value by their own roundings: half a step of
        # bf16 each (2^-8 of a value no larger than the largest in the cache), and the f16 weights' 2^-11 each
        assert float((part[39] - whole[39]).abs().max()) <= (2 * 2.0**-8 + 2 * 2.0**-10) * float(values.abs().max())
        assert bool((part[40:] == 5.0).all())
        mixed = make_batch(nb, torch, [3, 40, 2], [10, 3, 20], np.array([[0], [1], [0]]), **bounds)
        part.fill_(5.0)
        cache.attend(mixed, query, part, int32(torch, [1]), 64)
        with pytest.raises(nb.NeedleError) as e:
            cache.check()
        assert "sequence" in e.value.message
        assert bool((part[3:43] == 5.0).all()) and bool((part[45:] == 5.0).all()) and not bool((part[:3] == 5.0).any()) and not bool((part[43:45] == 5.0).any())


@pytest.mark.parametrize("bounds", [{"max_length": 0}, {"max_rows": 0}, {"max_rows": 0, "max_length": 0}, {"rows": 1}])
def test_bounds_below_what_the_sequences_have(nb, torch, bounds):
    """Nothing is written, and it is reported, with and without a prefix."""
    cache = nb.KvCache(2, 64, 4, device=0)
    x, y = (torch.ones(2, h, 64, dtype=torch.bfloat16, device="cuda:0") for h in (2, 4))
    for prefix in (0, 70):
        out = torch.full_like(y, 5.0)
        cache.attend(make_batch(nb, torch, [2], [2], np.array([[0]]), **bounds), y, out, int32(torch, [1, 2]), prefix)
        with pytest.raises(nb.NeedleError) as e:
            cache.check()
        assert "sequence" in e.value.message and bool((out == 5.0).all())
    cache.append(make_batch(nb, torch, [2], [2], np.array([[0]]), **bounds), x, x)
    with pytest.raises(nb.NeedleError):
        cache.check()


def test_attend_in_place(nb, torch):
    """The output may be the query itself: every row and head is read before it is written."""
    rng = np.random.default_rng(59)
    cache = nb.KvCache(2, 64, 80, device=0)
    keys, values = (random_rows(rng, torch, 5000, 2, 64, torch.bfloat16) for _ in range(2))
    cache.append(make_batch(nb, torch, [5000], [5000], np.arange(79)[None]), keys, values)
    for n, length, prefix in ((1, 5, 100), (40, 300, 1000), (1, 5000, 0), (600, 5000, 2000)):
        query = random_rows(rng, torch, n, 8, 64, torch.bfloat16)
        batch = make_batch(nb, torch, [n], [length], np.arange(79)[None])
        want = torch.empty_like(query)
        cache.attend(batch, query, want, int32(torch, range(79)), prefix)
        cache.attend(batch, query, query, int32(torch, range(79)), prefix)
        assert torch.equal(query, want)
    cache.check()


def test_attend_is_the_same_every_time(nb, torch):
    a, b = (attend_case(nb, torch, 47, [3] * 50, [100 + i for i in range(50)], 900, 8, 2, 128, "int8", "bf16") for _ in range(2))
    assert torch.equal(a, b)


def test_attend_refuses(nb, torch):
    cache = nb.KvCache(2, 64, 8, device=0)
    batch = make_batch(nb, torch, [2], [2], np.array([[0]]))
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda:0")
    ok = torch.zeros_like(q)
    with pytest.raises(nb.NeedleError):
        cache.attend(batch, q[:, :3], ok[:, :3])  # heads not a multiple
    with pytest.raises(nb.NeedleError):
        cache.attend(batch, q.float(), ok.float())
    with pytest.raises(nb.NeedleError):
        cache.attend(batch, q, ok.half())
    with pytest.raises(nb.NeedleError):
        cache.attend(batch, q, ok[:1].expand(2, 4, 64))  # rows of the output overlap
    with pytest.raises(ValueError):
        cache.attend(batch, q, ok, None, 0) if False else cache.attend(batch, q[:1], ok)
    with pytest.raises(ValueError):
        cache.attend(batch, q, ok, int32(torch, [1]), 65)
    with pytest.raises(ValueError):
        cache.append(batch, torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))
    from rustyneedle_b200 import serving

    L = serving._library()
    rows = serving.nb_rows(q.data_ptr(), 2, 256, 64)
    need = ctypes.c_size_t()
    assert L.nb_kv_cache_attend_workspace(cache._h, batch._ref, 0, 4, ctypes.byref(need)) == 0 and need.value > 0
    assert L.nb_kv_cache_attend(cache._h, batch._ref, None, 0, rows, rows, 4, 1.0, None, 0, None) == -4
    space = torch.zeros(need.value + 64, dtype=torch.uint8, device="cuda:0")
    assert L.nb_kv_cache_attend(cache._h, batch._ref, None, 0, rows, rows, 4, 1.0, space.data_ptr(), need.value - 1, None) == -4
    assert L.nb_kv_cache_attend(cache._h, batch._ref, None, 0, rows, rows, 4, 1.0, space.data_ptr() + 4, need.value, None) == -4
    assert L.nb_kv_cache_attend(cache._h, batch._ref, None, 65, rows, rows, 4, 1.0, space.data_ptr(), need.value, None) == -4
    negative = serving.nb_rows(q.data_ptr(), 2, -256, 64)
    assert L.nb_kv_cache_append(cache._h, batch._ref, negative, rows, None) == -4
    assert L.nb_kv_cache_append(cache._h, batch._ref, rows, serving.nb_rows(q.data_ptr(), 1, 256, 64), None) == -4
    cache.check()


def test_broadcast_inputs(nb, torch):
    """Strides of zero: one row of keys for all rows, one query for all heads."""
    rng = np.random.default_rng(48)
    rows, lengths, table = [4], [4], np.array([[0]])
    cache = nb.KvCache(2, 64, 1, device=0)
    keys = random_rows(rng, torch, 1, 2, 64, torch.float16).expand(4, 2, 64)
    values = random_rows(rng, torch, 4, 1, 64, torch.float16).expand(4, 2, 64)
    cache.append(make_batch(nb, torch, rows, lengths, table), keys, values)
    query = random_rows(rng, torch, 4, 1, 64, torch.float16).expand(4, 4, 64)
    check_attend(nb, torch, cache, query, keys, values, rows, lengths, table, out=torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda:0"))


def test_nothing_to_do(nb, torch):
    cache = nb.KvCache(2, 64, 1, device=0)
    empty = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    for rows, lengths in (([], []), ([0, 0], [0, 3])):
        table = np.zeros((len(rows), 1), dtype=np.int32)
        batch = make_batch(nb, torch, rows, lengths, table)
        cache.append(batch, empty, empty)
        cache.read(batch, empty, empty)
        cache.attend(batch, empty, empty)
    cache.check()


# ---------------------------------------------------------------------------------------------- streams, graphs, threads


def test_captured_step_follows_its_arrays_and_two_graphs_share_nothing(nb, torch):
    """Append and attend, captured twice, replayed on two streams at once with lengths that grow between replays."""
    rng = np.random.default_rng(50)
    kv, dim, heads, prefix = 2, 64, 4, 300
    lengths0 = [60, 1, 127]
    prefix_pages, table, pages = paged(rng, [t + 70 for t in lengths0] * 2, -(-prefix // PAGE))
    cache = nb.KvCache(kv, dim, pages, device=0)
    pk, pv = (random_rows(rng, torch, prefix, kv, dim, torch.bfloat16) for _ in range(2))
    cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), pk, pv)
    shared = int32(torch, prefix_pages)
    sides = []
    for side in range(2):
        own = table[side * 3 : side * 3 + 3]
        tk, tv = (random_rows(rng, torch, sum(lengths0), kv, dim, torch.bfloat16) for _ in range(2))
        cache.append(make_batch(nb, torch, lengths0, lengths0, own), tk, tv)
        lengths = int32(torch, lengths0)
        batch = nb.KvBatch(int32(torch, [0, 1, 2, 3]), lengths, int32(torch, own), rows=3, max_rows=1, max_length=200)
        k, v = (torch.zeros(3, kv, dim, dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
        q = torch.zeros(3, heads, dim, dtype=torch.bfloat16, device="cuda:0")
        out = torch.zeros_like(q)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            lengths.add_(1)
            cache.append(batch, k, v)
            cache.attend(batch, q, out, shared, prefix)
        sides.append(dict(batch=batch, own=own, tk=tk, tv=tv, k=k, v=v, q=q, out=out, graph=graph, stream=torch.cuda.Stream(), news=[]))
    for step in range(5):
        for s in sides:
            new = [random_rows(rng, torch, 3, h, dim, torch.bfloat16) for h in (kv, kv, heads)]
            s["news"].append(new)
            s["k"].copy_(new[0]), s["v"].copy_(new[1]), s["q"].copy_(new[2])
        torch.cuda.synchronize()
        for s in sides:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
    cache.check()
    for s in sides:
        first, keys, values = 0, [pk], [pv]
        for b, t in enumerate(lengths0):
            keys += [s["tk"][first : first + t]] + [n[0][b : b + 1] for n in s["news"]]
            values += [s["tv"][first : first + t]] + [n[1][b : b + 1] for n in s["news"]]
            first += t
        got = s["out"].clone()
        want = check_attend(nb, torch, cache, s["news"][-1][2], torch.cat(keys), torch.cat(values), [1, 1, 1], [t + 5 for t in lengths0], s["own"], prefix, shared)
        # the plan's split depends on the bounds alone: an eager call with closer bounds may round the last bit otherwise
        assert float((got.float() - want.float()).abs().max()) <= 2.0**-7 * float(want.float().abs().max())


def test_calls_on_another_stream_and_from_threads(nb, torch):
    import threading

    rng = np.random.default_rng(51)
    cache = nb.KvCache(2, 64, 40, device=0)
    jobs, failures = [], []
    for side in range(4):
        table = np.arange(side * 10, side * 10 + 10)[None]
        keys, values = (random_rows(rng, torch, 600, 2, 64, torch.float16) for _ in range(2))
        jobs.append((table, keys, values, random_rows(rng, torch, 5, 4, 64, torch.float16)))
    torch.cuda.synchronize()

    def work(table, keys, values, query):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                whole = make_batch(nb, torch, [600], [600], table)
                batch = make_batch(nb, torch, [5], [600], table)
                out = torch.zeros_like(query)
                for _ in range(20):
                    cache.append(whole, keys, values)
                    cache.attend(batch, query, out)
                torch.cuda.current_stream().synchronize()
                check_attend(nb, torch, cache, query, keys, values, [5], [600], table)
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failures, failures[0]


def test_another_current_device(nb, torch):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    cache = nb.KvCache(2, 64, 4, device=1)
    with torch.cuda.device(0):
        keys = torch.randn(3, 2, 64, device="cuda:1")
        batch = nb.KvBatch(int32(torch, [0, 3], "cuda:1"), int32(torch, [3], "cuda:1"), int32(torch, [[2]], "cuda:1"), rows=3, max_rows=3, max_length=3)
        out = torch.empty_like(keys)
        cache.append(batch, keys, keys)
        cache.read(batch, out, torch.empty_like(out))
        assert torch.cuda.current_device() == 0
        assert np.array_equal(numbers(out), held(numbers(keys), "int8", torch.float32, torch))


# -------------------------------------------------------------------------------------------------------------- verify


def verify_inputs(rng, torch, n, k, vocab, dtype, masked=False, given=True, temperature=1.0, noise=0.7):
    exact = rng.standard_normal((n, k + 1, vocab)) * 2 - 1.5 * rng.exponential(1.0, (n, k + 1, vocab))
    np.put_along_axis(exact, rng.integers(0, vocab, (n, k + 1, 1)), rng.uniform(4, 14, (n, k + 1, 1)), 2)
    logits = torch.tensor(exact, dtype=torch.float32).to(dtype_of(torch, dtype)).cuda()
    mask = None
    drafted = exact + noise * rng.standard_normal(exact.shape)
    if masked:
        allowed = rng.random((n, k + 1, vocab)) < 0.3
        allowed[rng.random((n, k + 1)) < 0.1] = False
        words = -(-vocab // 32)
        padded = np.zeros((n, k + 1, words * 32), dtype=np.uint8)
        padded[..., :vocab] = allowed
        mask = np.packbits(padded, axis=-1, bitorder="little").view(np.uint32).reshape(n, k + 1, words)
        drafted = np.where(allowed | ~allowed.any(-1, keepdims=True), drafted, -np.inf)
    q = np.exp((drafted - drafted.max(-1, keepdims=True)) / (temperature or 1.0))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)[:, :k]
    tokens = np.zeros((n, k), dtype=np.int64)
    for b in range(n):
        for i in range(k):
            p = q[b, i].astype(np.float64)
            tokens[b, i] = drafted[b, i].argmax() if temperature == 0 else rng.choice(vocab, p=p / p.sum())
    accept, sample = rng.random((n, k)).astype(np.float32), rng.random(n).astype(np.float32)
    return dict(logits=logits, tokens=tokens, accept=accept, sample=sample, q=q if given else None, mask=mask, temperature=temperature)


def check_verify(nb, torch, x, counts=None):
    n, rows, vocab = x["logits"].shape
    cuda = lambda a, t: None if a is None else torch.tensor(np.ascontiguousarray(a), device="cuda:0").to(t)  # noqa: E731
    tokens, accepted = nb.verify_drafts(
        x["logits"], cuda(x["tokens"], torch.int32), cuda(x["accept"], torch.float32), cuda(x["sample"], torch.float32),
        draft_probabilities=cuda(x["q"], torch.float32), draft_counts=cuda(counts, torch.int32),
        mask_bits=None if x["mask"] is None else torch.tensor(x["mask"].view(np.int32), device="cuda:0"), temperature=x["temperature"])
    want = ref.verify(x["logits"].float().cpu().numpy(), x["tokens"], x["accept"], x["sample"], x["q"], counts, x["mask"], x["temperature"])
    assert np.array_equal(accepted.cpu().numpy(), want[1])
    assert np.array_equal(tokens.cpu().numpy(), want[0])
    return tokens, accepted


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 500, 4096, 8192, 20011])
@pytest.mark.parametrize("drafts", [0, 1, 4, 9])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_verify(nb, torch, vocab, drafts, dtype):
    rng = np.random.default_rng(vocab * 31 + drafts)
    n = 3 if vocab > 10000 else 17
    for masked, given, temperature in ((False, True, 1.0), (True, True, 0.7), (False, False, 1.3), (True, False, 0.0)):
        x = verify_inputs(rng, torch, n, drafts, vocab, dtype, masked, given, temperature)
        check_verify(nb, torch, x, rng.integers(-1, drafts + 2, n))
        check_verify(nb, torch, x)


@pytest.mark.parametrize("n", [1, 5, 160, 400])
def test_verify_batches(nb, torch, n):
    rng = np.random.default_rng(n)
    check_verify(nb, torch, verify_inputs(rng, torch, n, 3, 700, "bf16", True))
    check_verify(nb, torch, verify_inputs(rng, torch, min(n, 5), 2, 150001, "fp32"))


def test_verify_strange_logits(nb, torch):
    rng = np.random.default_rng(60)
    x = verify_inputs(rng, torch, 12, 2, 300, "fp32")
    l = x["logits"]
    l[0, 0, 5], l[1, 0], l[2, 0] = float("nan"), float("nan"), float("-inf")
    l[3, 0, 7] = float("inf")
    l[3, 0, 9] = float("inf")
    l[4, 1] = float("-inf")
    l[5] = 0.0
    l[6, :, 1:] = float("-inf")
    l[7] = 3.0e38
    l[8] = -3.0e38
    l[9, 0, :150] = -3.4e38
    x["tokens"][10] = [300, 2**31 - 1]
    x["tokens"][11] = [-1, 5]
    tokens, accepted = check_verify(nb, torch, x)
    assert tokens[1].tolist() == [-1, -1, -1] and tokens[2].tolist() == [-1, -1, -1] and accepted[10] == 0 and accepted[11] == 0
    x["temperature"] = 0.0
    check_verify(nb, torch, x)
    x["temperature"] = 1e-30
    check_verify(nb, torch, x)
    x["temperature"] = 1e30
    check_verify(nb, torch, x)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_verify_logits_masked_with_the_lowest_value(nb, torch, dtype, temperature):
    """Masks written into the logits: the type's lowest value, -inf, both, in all places but one and in all."""
    rng = np.random.default_rng(65)
    x = verify_inputs(rng, torch, 9, 2, 517, dtype, temperature=temperature)
    l = x["logits"]
    low = torch.finfo(l.dtype).min
    drop = torch.tensor(rng.random(l.shape) < 0.7, device="cuda:0")
    drop[2], drop[3], drop[6] = True, True, True
    drop[3, :, 400] = False
    l[:4] = torch.where(drop[:4], torch.full_like(l[:4], low), l[:4])
    l[4:7] = torch.where(drop[4:7], torch.full_like(l[4:7], float("-inf")), l[4:7])
    l[7, :, ::2], l[7, :, 1::2] = low, float("-inf")
    l[8], l[8, 0, 3] = low, torch.finfo(l.dtype).max
    check_verify(nb, torch, x)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_verify_greedy_takes_the_lowest_of_equal_maxima(nb, torch, dtype):
    """Equal maxima, infinities behind NaNs, rows of NaN or -inf alone, in rows long enough for every thread's steps."""
    rng = np.random.default_rng(67)
    for vocab in (40000, 40011):
        x = verify_inputs(rng, torch, 8, 3, vocab, dtype, given=False, temperature=0.0)
        l = x["logits"]
        top = torch.finfo(l.dtype).max
        l[0, :, 777] = l[0, :, 30001] = 60.0
        l[1, :, 5000] = l[1, :, 20000] = float("inf")
        l[1, :, 4990:5000] = float("nan")
        l[2, :, 9] = float("nan")
        l[2, :, 100] = l[2, :, 39999] = top
        l[2, :, 35000] = float("inf")
        l[3] = float("nan")
        l[3, 0, 39990] = -5.0
        l[4] = float("-inf")
        l[4, 0, 12345] = torch.finfo(l.dtype).min
        l[5] = 0.0
        l[6] = -0.0
        l[6, :, 3333] = 0.0
        l[7, :, 1:] = torch.sort(l[7, :, 1:], dim=-1).values  # the maximum grows with every step
        x["tokens"][:] = l[:, :3].float().nan_to_num(nan=float("-inf"), posinf=float("inf")).argmax(-1).cpu().numpy()
        check_verify(nb, torch, x)


@pytest.mark.parametrize("drafts", [63, 64, 65, 130])
def test_verify_many_drafts(nb, torch, drafts):
    """More drafts than a block holds at once, with runs that are accepted to the end and runs that are not."""
    rng = np.random.default_rng(66)
    for given, temperature in ((True, 1.0), (False, 1.0), (False, 0.0)):
        x = verify_inputs(rng, torch, 5, drafts, 130, "fp32", given=given, temperature=temperature, noise=0.05)
        if given:
            x["accept"] *= 0.9
        else:
            x["accept"][:3] = 0.0
        if temperature == 0:
            x["tokens"][:3] = x["logits"][:3, :drafts].argmax(-1).cpu().numpy()
        counts = [drafts, drafts - 1, min(drafts, 64), drafts, 0]
        check_verify(nb, torch, x)
        check_verify(nb, torch, x, np.array(counts, dtype=np.int32))


def test_verify_uniforms_at_their_ends(nb, torch):
    rng = np.random.default_rng(61)
    for given in (True, False):
        x = verify_inputs(rng, torch, 40, 2, 333, "fp32", given=given)
        x["sample"][:10], x["sample"][10:20] = 0.0, np.float32(1 - 2.0**-24)
        x["accept"][:5], x["accept"][5:25] = 0.0, np.float32(1 - 2.0**-24)
        x["sample"][20:24] = [1.0, 2.0, -1.0, np.nan]
        x["accept"][30:32] = np.nan
        check_verify(nb, torch, x)


def test_verify_draft_equal_to_the_target(nb, torch):
    """q = p in 32 bits: nothing or nearly nothing is left above the draft, also for an accept number that cannot be met."""
    rng = np.random.default_rng(62)
    x = verify_inputs(rng, torch, 30, 3, 100, "fp32", noise=0.0)
    x["accept"][:] = 2.0
    check_verify(nb, torch, x)
    x["q"][:] = 1.0  # p nowhere exceeds q: the draw is from p
    check_verify(nb, torch, x)


def test_verify_strided_rows_and_given_outputs(nb, torch):
    rng = np.random.default_rng(63)
    x = verify_inputs(rng, torch, 4, 2, 1001, "bf16")
    room = torch.full((4, 3, 1013), float("inf"), dtype=torch.bfloat16, device="cuda:0")
    room[..., 5:1006] = x["logits"]
    x["logits"] = room[..., 5:1006]
    check_verify(nb, torch, x)
    with pytest.raises(ValueError):
        nb.verify_drafts(room[:, :2, :1001], *[torch.zeros(1)] * 3)


def test_verify_graph_replays_with_new_numbers(nb, torch):
    rng = np.random.default_rng(64)
    xs = [verify_inputs(rng, torch, 6, 3, 5000, "fp32") for _ in range(3)]
    put = lambda x: [x["logits"].clone()] + [torch.tensor(x[k], device="cuda:0").to(torch.int32 if k == "tokens" else torch.float32) for k in ("tokens", "accept", "sample", "q")]  # noqa: E731
    held_ = put(xs[0])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tokens, accepted = nb.verify_drafts(held_[0], held_[1], held_[2], held_[3], held_[4])
    for x in xs:
        [a.copy_(b) for a, b in zip(held_, put(x))]
        graph.replay()
        torch.cuda.synchronize()
        want = ref.verify(x["logits"].cpu().numpy(), x["tokens"], x["accept"], x["sample"], x["q"])
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(accepted.cpu().numpy(), want[1])


# ---------------------------------------------------------------------------------------------------------- together


def test_a_drafted_step_over_a_shared_prompt(nb, torch):
    """One attention layer with a vocabulary, decoded with drafts: append the drafted rows, attend, verify; then the next
    step appends over the rejected rows. Greedy drafted decoding has to give the tokens that plain decoding gives."""
    rng = np.random.default_rng(70)
    kv, heads, dim, vocab, prefix, n, drafts = 2, 4, 64, 257, 150, 6, 3
    width = heads * dim
    to = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda:0")  # noqa: E731
    embed = to(rng.standard_normal((vocab, width)))
    wq, wk, wv = to(rng.standard_normal((width, width)) / 16), to(rng.standard_normal((width, kv * dim)) / 16), to(rng.standard_normal((width, kv * dim)) / 16)
    head = to(rng.standard_normal((width, vocab)))

    def project(ids):
        x = embed[ids]
        return x, (x @ wq).view(-1, heads, dim).bfloat16(), (x @ wk).view(-1, kv, dim).bfloat16(), (x @ wv).view(-1, kv, dim).bfloat16()

    prompt = torch.tensor(rng.integers(0, vocab, prefix), device="cuda:0")
    first = rng.integers(0, vocab, n)

    def decode(with_drafts, steps):
        pages = 3 + n * 2
        cache = nb.KvCache(kv, dim, pages, device=0)
        shared = int32(torch, [0, 1, 2])
        table = (3 + np.arange(n * 2)).reshape(n, 2)
        _, _, k, v = project(prompt)
        cache.append(nb.KvBatch(int32(torch, [0, prefix]), int32(torch, [prefix]), shared[None], rows=prefix, max_rows=prefix, max_length=prefix), k, v)
        text = [[int(t)] for t in first]
        count = drafts if with_drafts else 0
        taken = 0
        while min(len(t) for t in text) <= steps:
            guess = rng.integers(0, vocab, (n, count))
            if with_drafts:  # half of the guesses are what plain decoding says
                for b in range(n):
                    for i in range(count):
                        at = len(text[b]) + i
                        if at < len(plain[b]) and rng.random() < 0.7:
                            guess[b, i] = plain[b][at]
            ids = np.concatenate([np.array([t[-1] for t in text])[:, None], guess], 1)
            x, q, k, v = project(torch.tensor(ids.ravel(), device="cuda:0"))
            lengths = [len(t) + count for t in text]
            batch = make_batch(nb, torch, [count + 1] * n, lengths, table)
            cache.append(batch, k, v)
            out = torch.empty_like(q)
            cache.attend(batch, q, out, shared, prefix)
            logits = ((x + out.view(-1, width).float()) @ head).view(n, count + 1, vocab).contiguous()
            tokens, accepted = nb.verify_drafts(logits, int32(torch, guess).view(n, count), None, None, temperature=0.0)
            for b, row in enumerate(tokens.cpu().tolist()):
                text[b] += [t for t in row if t >= 0]
            taken += int(accepted.sum())
        cache.check()
        return [t[: steps + 1] for t in text], taken

    plain, _ = decode(False, 40)
    drafted, taken = decode(True, 40)
    assert taken > n * 10
    assert drafted == plain
