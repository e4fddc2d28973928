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
