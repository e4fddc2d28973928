"""Drafted decoding, what needs no GPU: rules that the kernels' sources keep and
arguments at their limits."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustyneedle_b200", "csrc")


def _kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for body in text.split("__global__")[1:]:
            yield os.path.basename(path), body


def test_no_kernel_reaches_into_a_cluster_before_all_of_it_runs():
    """Another CTA's shared memory may be touched once that CTA is known to run: a cluster barrier comes before the first
    remote access of every kernel that makes one."""
    seen = set()
    for name, body in _kernels():
        first = body.find("map_shared_rank")
        if first < 0:
            continue
        seen.add(name)
        barriers = [body.find(word) for word in ("cluster_wait()", "cluster.sync()") if word in body]
        assert barriers and min(barriers) < first, name
    assert "verify.cu" in seen


@pytest.mark.parametrize("name", ["kv_heads", "head_dim", "pages"])
@pytest.mark.parametrize("value", [-1, 1 << 32, (1 << 32) + 4])
def test_cache_sizes_that_32_bits_do_not_hold_are_refused(native_built, name, value):
    import rustyneedle_b200 as nb

    with pytest.raises(ValueError, match=name):
        nb.KvCache(**{"kv_heads": 4, "head_dim": 64, "pages": 8, name: value})


class _Gpu:
    """What KvBatch asks of a tensor, without one."""

    device = type("Device", (), {"index": 0})

    def __init__(self, *shape):
        import torch

        self.shape, self.dtype, self.is_cuda = shape, torch.int32, True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape[0]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("name", ["rows", "max_rows", "max_length"])
@pytest.mark.parametrize("value", [-1, -(1 << 32) + 1, 1 << 32, (1 << 32) + 1])
def test_batch_bounds_that_32_bits_do_not_hold_are_refused(native_built, name, value):
    import rustyneedle_b200 as nb

    arrays = _Gpu(3), _Gpu(2), _Gpu(2, 1)
    nb.KvBatch(*arrays, rows=2, max_rows=1, max_length=9)
    with pytest.raises(ValueError, match=name):
        nb.KvBatch(*arrays, **{"rows": 2, "max_rows": 1, "max_length": 9, name: value})


@pytest.mark.parametrize("value", [-1, -(1 << 32) + 5, (1 << 32) + 5])
def test_a_prefix_length_that_32_bits_do_not_hold_is_refused(native_built, value):
    """Its lower 32 bits would name pages that prefix_pages does not hold."""
    import torch

    import rustyneedle_b200 as nb

    cache = object.__new__(nb.KvCache)
    cache._h, cache.device, cache.kv_heads, cache.head_dim = None, -1, 2, 64  # -1: tensors of the CPU
    batch = nb.KvBatch(_Gpu(2), _Gpu(1), _Gpu(1, 1), rows=1, max_rows=1, max_length=9)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="prefix_length"):
        cache.attend(batch, x, x, _Gpu(1), value)
