"""The operators that edit a paged cache (include/rlh_cache.h) where their
kernels go on for long or reach a limit, against the 64-bit forms of
tests/cache_ref.py."""
import numpy as np
import pytest
import torch

import rlh
import serve_ref as ref
from test_gpu_cache import run_move, word

pytestmark = pytest.mark.gpu


# ---- moving rows ------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
def test_move_of_more_lists_than_slices_fit(dim):
    """65535 sequences of 32 KV heads, lists past 256 entries: a launch of slices
    would hold 2^32 threads. Three sequences have rows to move."""
    n, kv, live = 65535, 32, (0, 40001, 65534)
    lengths = [300 if s in live else 0 for s in range(n)]
    b = ref.Batch([(0, x) for x in lengths], kv, dim, 16, rlh.F16, seed=dim, pad_rows=1)
    r = np.random.default_rng(dim)
    index, count = np.zeros((n, 1, 260), np.int32), np.zeros(n, np.int64)
    for s in live:
        index[s, 0] = np.sort(r.choice(300, 260, replace=False))
        count[s] = 260
    k, v = b.k.clone(), b.v.clone()
    for s in live:
        src, dst = index[s, 0], np.arange(260)
        for old, new in ((b.k, k), (b.v, v)):
            new[[b.page_of(s, j) for j in dst], :, dst % 16] = old[[b.page_of(s, int(j)) for j in src], :, src % 16]
    st = word()
    run_move(b, index, count, per_head=False, status=st, max_count=260)
    assert int(st) == 0
    assert torch.equal(b.k, k) and torch.equal(b.v, v)
