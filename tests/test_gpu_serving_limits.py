"""Drafted decoding on the GPU at the limits of what its calls allow, against
plain 64-bit forms."""

import numpy as np
import pytest

from tests import serving_reference as ref
from tests.test_gpu_serving import nb, torch, verify_inputs  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def cuda_inputs(torch, x):  # noqa: F811
    """verify_drafts' arguments for verify_inputs' numbers."""
    put = lambda a, t: None if a is None else torch.tensor(np.ascontiguousarray(a), device="cuda:0").to(t)  # noqa: E731
    args = [x["logits"], put(x["tokens"], torch.int32), put(x["accept"], torch.float32), put(x["sample"], torch.float32)]
    more = {"draft_probabilities": put(x["q"], torch.float32), "temperature": x["temperature"]}
    if x["mask"] is not None:
        more["mask_bits"] = torch.tensor(x["mask"].view(np.int32), device="cuda:0")
    return args, more


def plain(x, counts=None):
    return ref.verify(x["logits"].float().cpu().numpy(), x["tokens"], x["accept"], x["sample"], x["q"], counts, x["mask"], x["temperature"])


def test_verify_many_clusters_on_several_streams(nb, torch):  # noqa: F811
    """Clusters of one to eight blocks that start while others run: no block reaches into one that does not run yet."""
    rng = np.random.default_rng(80)
    jobs = []
    for n, vocab, temperature in ((3, 9001, 1.0), (70, 3000, 1.0), (160, 2100, 0.0), (300, 1500, 0.9), (600, 300, 1.0)):
        x = verify_inputs(rng, torch, n, 2, vocab, "bf16", temperature=temperature)
        jobs.append((cuda_inputs(torch, x), plain(x), torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(10):
        for (args, more), _, stream, got in jobs:
            with torch.cuda.stream(stream):
                got.append(nb.verify_drafts(*args, **more))
    torch.cuda.synchronize()
    for _, want, _, got in jobs:
        for tokens, accepted in got:
            assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(accepted.cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n, vocab", [(200, 50257), (64, 32000), (8, 129283), (600, 17001)])
def test_verify_greedy_passes_over_nan_in_long_rows(nb, torch, dtype, n, vocab):  # noqa: F811
    """Rows long enough for several full steps of every thread: all of them NaN, NaN in all places of some threads, NaN
    behind the maximum and before it, and infinities among them."""
    from tests.test_gpu_serving import dtype_of

    g = torch.Generator("cuda").manual_seed(vocab)
    kinds, drafts, nan, inf = 8, 1, float("nan"), float("inf")
    one = torch.randn(kinds, drafts + 1, vocab, generator=g, device="cuda:0")
    ids = torch.arange(vocab, device="cuda:0")
    lanes = (ids // 8 % 32 >= 5) & (ids // 8 % 32 <= 7)  # whole 16-byte pieces of one lane of every warp, however they start
    one[0] = nan
    one[1, :, lanes] = nan
    one[2, :, 3] = 50.0
    one[2, :, 9:] = nan
    one[3, :, : vocab - 7] = nan
    one[4, 0] = nan
    one[4, 0, vocab // 2] = -3.0
    one[5, :, vocab // 3 :] = nan
    one[5, :, vocab // 5] = inf
    one[6] = torch.where(lanes, nan, -inf)
    one = one.to(dtype_of(torch, dtype))
    clean = one.float().nan_to_num(nan=-inf, posinf=inf, neginf=-inf)
    x = dict(logits=one, tokens=clean[:, :drafts].argmax(-1).cpu().numpy(), accept=None, sample=None, q=None, mask=None, temperature=0.0)
    want = plain(x)
    assert (want[0][[0, 6]] == -1).all()
    of = torch.arange(n, device="cuda:0") % kinds
    tokens, accepted = nb.verify_drafts(one[of].contiguous(), torch.tensor(x["tokens"], dtype=torch.int32, device="cuda:0")[of].contiguous(), None, None, temperature=0.0)
    of = of.cpu().numpy()
    assert np.array_equal(tokens.cpu().numpy(), want[0][of]) and np.array_equal(accepted.cpu().numpy(), want[1][of])


def test_attend_with_a_bound_of_rows_beyond_the_batch(nb, torch):  # noqa: F811
    """max_rows may be as loose as the call allows: 2^26 rows of 64 heads are more (row, head) pairs than 31 bits count, and
    the launch follows the batch's own rows instead."""
    from tests.test_gpu_serving import attend_case

    for seed, rows, lengths, prefix, heads, kv in ((81, [3, 1], [40, 70], 100, 64, 1), (82, [20, 0, 5], [20, 3, 90], 0, 64, 1), (83, [2], [2], 65, 8, 2)):
        attend_case(nb, torch, seed, rows, lengths, prefix, heads, kv, 64, "int8", "bf16", bounds={"rows": sum(rows), "max_rows": 1 << 26})


@pytest.mark.parametrize("score", [10.0, 14.0, 25.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bounds", [{}, {"rows": 8192, "max_rows": 2048, "max_length": 1 << 14}, {"rows": 4000, "max_rows": 150, "max_length": 1 << 17}])
def test_attend_to_value_rows_of_zeros(nb, torch, kind, dim, score, bounds):  # noqa: F811
    """A position that draws most of the attention and gives nothing, written as zeros or never written: the small rest is as
    exact as without it. The bound is check_attend's, with its largest p vs over the rows that give something (a row of
    zeros counts with the smallest scale, 2^-60)."""
    from tests.test_gpu_serving import int32, make_batch, numbers, paged, random_rows

    rng = np.random.default_rng(int(score) + dim)
    kv, heads, prefix, rows, lengths = 2, 4, 300, [3, 40], [200, 230]
    prefix_pages, table, pages = paged(rng, lengths, -(-prefix // 64))
    total = prefix + sum(lengths)
    keys = random_rows(rng, torch, total, kv, dim, torch.bfloat16) * 0.2
    values = (0.02 + 0.004 * torch.randn(total, kv, dim, generator=torch.Generator("cuda").manual_seed(5), device="cuda:0")).to(torch.bfloat16)
    query = random_rows(rng, torch, bounds.get("rows", sum(rows)), heads, dim, torch.bfloat16) * 0.2
    # all other positions lie below the two rows of zeros, and those that were never written, by about `score`
    query[:, :, 0] = dim**0.5
    keys[:, :, 0] = -score
    written = torch.ones(total, dtype=torch.bool)
    zeros = [7, prefix + 20, prefix + lengths[0] + 64]
    keys[zeros] = 0
    values[zeros] = 0
    fresh = slice(prefix + lengths[0], prefix + lengths[0] + 64)  # the second sequence's first page
    keys[fresh], values[fresh], written[fresh] = 0, 0, False
    cache = nb.KvCache(kv, dim, pages, format=kind, device=0)
    cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), keys[:prefix], values[:prefix])
    own = written[prefix:].cuda()
    cache.append(make_batch(nb, torch, [lengths[0], lengths[1] - 64], lengths, table), keys[prefix:][own], values[prefix:][own])
    out = torch.full_like(query, 3.0)
    cache.attend(make_batch(nb, torch, rows, lengths, table, **bounds), query, out, int32(torch, prefix_pages), prefix)
    cache.check()
    kc, ks = ref.quantise(numbers(keys), kind)
    vc, vs = ref.quantise(numbers(values), kind)
    vs = np.where((vc == 0).all(-1), 2.0**-60, vs)
    n = sum(rows)
    want, mass, size, least = ref.attend(numbers(query[:n]), kc * ks[..., None], vc, vs, rows, lengths, prefix, dim**-0.5)
    weight = 2 * ((dim + 8) * 2.0**-23 * size + 2.0**-20)
    eps = torch.finfo(torch.bfloat16).eps
    bound = eps / 2 * np.abs(want) + mass * (2.0**-11 + weight + ((prefix + max(lengths)) / 8 + 16) * 2.0**-23) + 2.0**-33 * least
    off = np.abs(numbers(out[:n]) - want)
    assert (off <= bound).all(), float((off / np.abs(want)).max())


def test_tensors_of_no_rows_whatever_their_strides(nb, torch):  # noqa: F811
    """torch.tensor gives an empty array strides of zero."""
    from tests.test_gpu_serving import make_batch

    empty = lambda *shape: torch.tensor(np.zeros(shape), dtype=torch.bfloat16, device="cuda:0")  # noqa: E731
    assert empty(0, 2, 64).stride() == (0, 0, 0)
    cache = nb.KvCache(2, 64, 1, device=0)
    for rows, lengths in (([], []), ([0, 0], [0, 3])):
        batch = make_batch(nb, torch, rows, lengths, np.zeros((len(rows), 1), dtype=np.int32))
        cache.append(batch, empty(0, 2, 64), empty(0, 2, 64))
        cache.read(batch, empty(0, 2, 64), empty(0, 2, 64))
        cache.attend(batch, empty(0, 4, 64), empty(0, 4, 64))
    cache.check()
    none = lambda *shape: torch.zeros(*shape, dtype=torch.float32, device="cuda:0")  # noqa: E731
    for drafts in (0, 2):
        tokens, accepted = nb.verify_drafts(empty(0, drafts + 1, 50), none(0, drafts).int(), none(0, drafts), none(0))
        assert tokens.shape == (0, drafts + 1) and accepted.shape == (0,)


OUT_OF_BOUNDS = [  # rows, lengths, bounds: each with one sequence that breaks a bound without a row of it below the batch's rows
    ([3, 3], [3, 3], {"rows": 3}), ([3, 0, 2], [3, 200, 2], {"max_length": 100}), ([3, 0, 2], [3, 65, 2], {"max_length": 1000}),
    ([2, 0], [2, -1], {}), ([4, 4], [4, 4], {"rows": 0}), ([0, 0], [5, 90], {"max_length": 64}), ([5] * 300 + [2], [5] * 301, {"rows": 1500}),
    ([2000, 7], [2000, 7], {"rows": 2000}),  # by blocks of 16 rows
]


@pytest.mark.parametrize("call", ["append", "read", "attend"])
@pytest.mark.parametrize("case", range(len(OUT_OF_BOUNDS)))
def test_sequences_that_break_a_bound_are_reported_by_every_call(nb, torch, call, case):  # noqa: F811
    from tests.test_gpu_serving import held, make_batch, numbers, random_rows

    rows, lengths, more = OUT_OF_BOUNDS[case]
    rng = np.random.default_rng(90 + case)
    n, kv, dim = sum(rows), 8, 64
    pages = [max(1, -(-t // 64)) for t in lengths]
    stride = 1 if max(lengths) < 1000 else max(pages)
    table = np.arange(len(rows) * stride).reshape(len(rows), stride)
    cache = nb.KvCache(kv, dim, table.size, device=0)
    keys, values = (random_rows(rng, torch, n, kv, dim, torch.float32) for _ in range(2))
    good = make_batch(nb, torch, rows, [max(r, min(t, 64)) if stride == 1 else t for r, t in zip(rows, lengths)], table)
    cache.append(good, keys, values)
    cache.check()
    batch = make_batch(nb, torch, rows, lengths, table, **more)
    out = [torch.full_like(keys, 9.0) for _ in range(2)]
    if call == "append":
        cache.append(batch, -keys, -values)
    elif call == "read":
        cache.read(batch, *out)
    else:
        cache.attend(batch, keys.bfloat16(), torch.full_like(keys, 9.0, dtype=torch.bfloat16))
    with pytest.raises(nb.NeedleError) as e:
        cache.check()
    assert e.value.status == -4 and "sequence" in e.value.message
    cache.check()  # cleared
    if call == "append":
        cache.read(good, *out)
        cache.check()
        keys = -keys
    if call != "attend":  # the others are served
        first = rows[0] if batch.rows else 0
        assert np.array_equal(numbers(out[0][:first]), held(numbers(keys[:first]), "int8", torch.float32, torch))
        left = out[0][batch.rows :]
        want = held(numbers(-keys[batch.rows :]), "int8", torch.float32, torch) if call == "append" else np.full(left.shape, 9.0)
        assert np.array_equal(numbers(left), want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n, drafts, vocab, masked, given, temperature", [
    (60, 9, 20011, False, False, 1.0), (200, 9, 8192, True, True, 0.8), (6, 9, 129283, False, True, 1.0), (400, 9, 5000, False, True, 1.3),
    (2, 9, 300007, False, False, 1.0), (30, 9, 300, True, False, 1.0), (20, 70, 500, True, True, 1.0), (20, 130, 90, False, True, 2.0)])
def test_verify_accept_numbers_next_to_their_border(nb, torch, dtype, n, drafts, vocab, masked, given, temperature):  # noqa: F811
    """The accept number is a step of f32 below p / q or above it, so that only a 64-bit p decides rightly: runs of drafts
    below it, then one above."""
    rng = np.random.default_rng(vocab)
    # the call takes an f32: 0.8 is 1.5e-8 above, which moves a p of e^-30 by 6e-7, ten steps of an accept number
    temperature = float(np.float32(temperature))
    x = verify_inputs(rng, torch, n, drafts, vocab, dtype, masked, given, temperature, noise=0.3)
    logits = x["logits"].double().cpu().numpy()
    for b in range(n):
        for i in range(drafts):
            l = logits[b, i]
            if masked and ref.unpack(x["mask"][b, i], vocab).any():
                l = np.where(ref.unpack(x["mask"][b, i], vocab), l, -np.inf)
            p = np.exp((l - l.max()) / temperature)
            p /= p.sum()
            d = int(x["tokens"][b, i])
            border = p[d] / (float(x["q"][b, i, d]) if given else 1.0)
            u = np.float32(border)
            above = b > 0 and (rng.random() < 1.5 / drafts or b == 1)
            if (float(u) > border) != above:
                u = np.nextafter(u, np.float32(np.inf if above else -np.inf))
            x["accept"][b, i] = u
    (args, more), want = cuda_inputs(torch, x), plain(x)
    tokens, accepted = nb.verify_drafts(*args, **more)
    assert want[1][0] == drafts and want[1][1] == 0
    assert np.array_equal(accepted.cpu().numpy(), want[1]), (accepted.cpu().numpy() != want[1]).mean()
    assert np.array_equal(tokens.cpu().numpy(), want[0])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bounds", [{}, {"rows": 8192, "max_rows": 2048, "max_length": 1 << 14}, {"rows": 4000, "max_rows": 150, "max_length": 1 << 17}])
@pytest.mark.parametrize("prefix, lengths", [(0, [30, 400, 9]), (700, [30, 400, 9]), (5000, [3000, 5, 60])])
def test_a_wait_of_the_attention_that_runs_out(nb, torch, bounds, dim, prefix, lengths):  # noqa: F811
    """The first block of every launch gives up: its rows are NaN, the others as they are without it, the call's status is
    a timeout, once, and the next call is whole again."""
    from rustyneedle_b200 import debug
    from tests.test_gpu_serving import int32, make_batch, paged, random_rows

    rng = np.random.default_rng(prefix + dim)
    kv, heads, rows = 2, 6, [3, 5, 1]
    prefix_pages, table, pages = paged(rng, lengths, -(-prefix // 64))
    cache = nb.KvCache(kv, dim, pages, device=0)
    keys, values = (random_rows(rng, torch, prefix + sum(lengths), kv, dim, torch.bfloat16) for _ in range(2))
    if prefix:
        cache.append(make_batch(nb, torch, [prefix], [prefix], prefix_pages[None]), keys[:prefix], values[:prefix])
    cache.append(make_batch(nb, torch, lengths, lengths, table), keys[prefix:], values[prefix:])
    query = random_rows(rng, torch, bounds.get("rows", sum(rows)), heads, dim, torch.bfloat16)
    batch, shared = make_batch(nb, torch, rows, lengths, table, **bounds), int32(torch, prefix_pages)

    def attend():
        out = torch.full_like(query, 3.0)
        cache.attend(batch, query, out, shared, prefix)
        return out

    whole = attend()
    cache.check()
    assert bool(torch.isfinite(whole).all())
    for _ in range(2):
        debug.expire_attention(cache, True)
        part = attend()
        debug.expire_attention(cache, False)
        with pytest.raises(nb.NeedleError) as e:
            cache.check()
        assert e.value.status == -9  # NB_ERR_TIMEOUT
        cache.check()
        lost = part.isnan()
        assert bool(lost[0, : heads // kv].all())  # the first tile is the first sequence's, or the batch's, of the first kv head
        assert not bool(lost[:, heads // kv :].any())
        assert torch.equal(torch.where(lost, whole, part), whole)
        if not prefix:
            assert not bool(lost[rows[0] :].any())
        assert torch.equal(attend(), whole)
        cache.check()


def test_a_report_names_all_that_was_met(nb, torch):  # noqa: F811
    """A wait that ran out, a sequence out of its bounds and a bad page in one report, none of them lost."""
    from rustyneedle_b200 import debug
    from tests.test_gpu_serving import int32, make_batch

    cache = nb.KvCache(2, 64, 4, device=0)
    x = torch.ones(6, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    batch = make_batch(nb, torch, [2, 2, 2], [2, 2, 70], np.array([[0, 1], [1, 0], [2, 9]]))
    bad = make_batch(nb, torch, [2, 2, 2], [2, 1, 70], np.array([[0, 1], [1, 0], [2, 9]]))
    for first, status, words in ((bad, -9, ["wait", "sequence", "page"]), (batch, -9, ["wait", "page"])):
        debug.expire_attention(cache, True)
        cache.attend(first, x, torch.empty_like(x), int32(torch, [3]), 10)
        debug.expire_attention(cache, False)
        with pytest.raises(nb.NeedleError) as e:
            cache.check()
        assert e.value.status == status and [w for w in ("wait", "sequence", "page") if w in e.value.message] == words
        cache.check()
    cache.append(bad, x, x)
    with pytest.raises(nb.NeedleError) as e:
        cache.check()
    assert e.value.status == -4 and "sequence" in e.value.message and "page" in e.value.message
    cache.check()
