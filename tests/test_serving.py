"""Drafted decoding, what needs no GPU: refusals of the C ABI, the pool's byte
order and the batch search, and the plain forms against themselves."""

import ctypes

import numpy as np
import pytest

from tests import serving_reference as ref


@pytest.fixture(scope="module")
def L(native_built):
    from rustyneedle_b200 import serving

    return serving._library()


def _message():
    from rustyneedle_b200._native import lib

    return lib().nb_last_error().decode()


@pytest.mark.parametrize("args, word", [
    ((0, 7, 4, 64, 8), "format"), ((0, 0, 0, 64, 8), "kv_heads"), ((0, 0, 257, 64, 8), "kv_heads"), ((0, 0, 4, 96, 8), "head_dim"),
    ((0, 1, 4, 64, 0), "page"),
])
def test_cache_create_refuses(L, args, word):
    h = ctypes.c_void_p()
    assert L.nb_kv_cache_create(*args, ctypes.byref(h)) == -4
    assert word in _message() and not h.value


def test_cache_create_needs_a_device_and_a_place(L):
    import torch

    assert L.nb_kv_cache_create(0, 0, 4, 64, 8, None) == -4
    if not torch.cuda.is_available():
        h = ctypes.c_void_p()
        assert L.nb_kv_cache_create(0, 0, 4, 64, 8, ctypes.byref(h)) == -10


def test_null_arguments_are_refused(L):
    from rustyneedle_b200 import serving

    n = ctypes.c_size_t()
    assert L.nb_kv_cache_append(None, None, None, None, None) == -4
    assert L.nb_kv_cache_read(None, None, None, None, None) == -4
    assert L.nb_kv_cache_attend(None, None, None, 0, None, None, 4, 1.0, None, 0, None) == -4
    assert L.nb_kv_cache_attend_workspace(None, None, 0, 4, ctypes.byref(n)) == -4
    assert L.nb_kv_cache_check(None, None) == -4
    assert L.nb_verify_drafts(0, None, None) == -4
    L.nb_kv_cache_release(None)
    assert serving.PAGE == 64


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1, row_stride=1 << 30), "vocab"), (dict(drafts=2000), "drafts"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=1e-38), "temperature"),
    (dict(row_stride=99), "row_stride"), (dict(logits=None), "needed"), (dict(draft_tokens=None), "draft_tokens"), (dict(tokens=None), "needed"),
    (dict(sample_uniforms=None), "uniforms"), (dict(accept_uniforms=None), "uniforms"), (dict(tokens=4098), "aligned"), (dict(logits=4097), "aligned"),
])
def test_verify_refuses_before_any_work(L, change, word):
    from rustyneedle_b200.serving import nb_verify

    args = dict(sequences=2, drafts=3, vocab=100, dtype=0, row_stride=100, logits=4096, draft_tokens=4096, accept_uniforms=4096, sample_uniforms=4096,
                temperature=1.0, tokens=4096, accepted=4096)
    args.update(change)
    a = nb_verify()
    for name, value in args.items():
        setattr(a, name, value)
    assert L.nb_verify_drafts(0, a, None) == -4
    assert word in _message()


@pytest.mark.parametrize("dim", [64, 128])
def test_every_value_code_has_its_own_byte(dim):
    p, d = np.meshgrid(np.arange(64), np.arange(dim), indexing="ij")
    at = (p // 16) * 16 * dim + (d // 32) * 512 + (d % 8) * 64 + (p % 16 // 4) * 16 + (d % 32 // 8) * 4 + p % 4
    assert sorted(at.ravel()) == list(range(64 * dim))


def _search(starts, row):
    """sequence_of (serving.cuh), a warp's steps written out."""
    lo, hi = 0, len(starts) - 1
    while hi - lo > 1:
        step = (hi - lo + 31) // 32
        probes = [lo + lane * step for lane in range(32)]
        below = [at < hi and starts[at] <= row for at in probes]
        k = max([i for i, x in enumerate(below) if x], default=0)
        lo += k * step
        hi = min(hi, lo + step)
    return lo


def test_search_finds_the_sequence_of_every_row():
    rng = np.random.default_rng(5)
    for n in (1, 2, 31, 32, 33, 64, 1000, 1025, 3000):
        rows = rng.integers(0, 4, n)
        rows[rng.random(n) < 0.3] = 0
        starts = np.concatenate([[0], np.cumsum(rows)])
        for row in range(starts[-1]):
            b = _search(starts, row)
            assert starts[b] <= row < starts[b + 1]


def test_search_stays_in_range_whatever_the_starts():
    rng = np.random.default_rng(6)
    for n in (1, 5, 40, 1500):
        for _ in range(50):
            starts = rng.integers(-(2**31), 2**31, n + 1)
            assert 0 <= _search(starts, int(rng.integers(0, 100))) < n


def test_plain_quantisation_rounds_halves_to_even():
    x = np.zeros((1, 64), dtype=np.float32)
    x[0, :6] = [127, 0.5, 1.5, 2.5, -0.5, -2.5]
    codes, scale = ref.quantise(x, "int8")
    assert scale[0] == 1.0 and list(codes[0, :6]) == [127, 0, 2, 2, 0, -2]
    y = np.array([448.0, 17.0, 19.0, 2.0**-10, 3 * 2.0**-10, 460.0])
    assert list(ref.e4m3(y)) == [448.0, 16.0, 20.0, 0.0, 2.0**-8, 448.0]


def test_plain_verification_follows_the_target():
    """With many uniforms, the first token of a verification is distributed as the target's softmax."""
    rng = np.random.default_rng(7)
    vocab, n = 5, 20000
    x = rng.standard_normal(vocab).astype(np.float32)
    q = np.exp(rng.standard_normal(vocab))
    q = (q / q.sum()).astype(np.float32)
    drafted = rng.choice(vocab, n, p=q / q.sum())[:, None]
    got, _ = ref.verify(np.broadcast_to(x, (n, 2, vocab)), drafted, rng.random((n, 1)), rng.random(n), np.broadcast_to(q, (n, 1, vocab)))
    p = np.exp(x) / np.exp(x).sum()
    share = np.bincount(got[:, 0], minlength=vocab) / n
    assert np.abs(share - p).max() < 5 * np.sqrt(0.25 / n)  # five standard deviations
