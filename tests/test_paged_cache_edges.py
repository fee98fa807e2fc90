"""The paged key-value cache at its edges: settings in which nothing is chosen, values that few bits lose, calls that
follow each other without a pause, ids of 64 bits, caches that share memory.

The oracles are those of test_paged_cache.py: the operators' definition in 64 bits, position by position.
"""
import numpy as np
import pytest
import torch

from test_paged_cache import dev, make_case, oracle_evict


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.gpu
@pytest.mark.parametrize("lens,page,init,local", [
    ([131072, 130999], 1, 64, 4096), ([300, 301, 5000, 0, 1], 1, 4, 6), ([409600], 1, 0, 1), ([65536, 100, 40000], 16, 1, 63),
    ([9000] * 70, 64, 3, 8), ([2000] * 300, 16, 0, 5)])
def test_eviction_to_the_first_and_last_pages(lens, page, init, local):
    """A budget that the first and the last pages fill: nothing is chosen, whatever the weights are and whatever the kernel
    before left on the chip (here all bits set, from a cache that is full of them)."""
    from unum_ops_b200 import evict_cache, paged_attention

    d = dev()
    rng = np.random.default_rng(len(lens) + lens[0])
    width = min(max(-(-n // page) for n in lens) + 1, 409600)
    table = rng.permutation(len(lens) * width).reshape(len(lens), width).astype(np.int32)
    w = rng.standard_normal((len(lens), 2, width * page)).astype(np.float32)
    w[..., ::7] = np.nan
    ln = np.array(lens, np.int32)
    args = [torch.from_numpy(x).to(d) for x in (table, ln, w)]
    want = oracle_evict(table, ln, w, init + local, init, local, page)
    q, kc, _, rows, n = [x.to(d) for x in make_case(3, [60000, 60000], 2, 16, 128, 1, "bf16")]
    kc.view(torch.int16).fill_(-1)
    for _ in range(10):
        paged_attention(q, kc, kc, rows, n)
        got = evict_cache(*args, budget=init + local, init_pages=init, local_pages=local, page_size=page)
        for name, x, y in zip(("table", "seqlens", "weights", "evicted"), got, want):
            np.testing.assert_array_equal(x.cpu().numpy(), y, err_msg=name)
