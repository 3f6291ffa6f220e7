"""Rotary positions, the paged cache in 16 bits and attention over shared prefixes at the edges of what their calls allow: the longest sequences, batches that change between replays, values and
scores at the ends of their types' ranges."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cache16_plain as plain  # noqa: E402
from test_cache16_gpu import as64, gen, near  # noqa: E402

pytestmark = pytest.mark.gpu

from calm_b200 import seqops  # noqa: E402


def test_a_sequence_of_as_many_tokens_as_an_int_holds():
    """Blocks of 21 tokens: the last one's threads count past 2^31.  (One row stands for all of them, the table has the first 32 positions.)"""
    cache, rot, n = seqops.Cache16.empty(4, 1, 16, 48, torch.float16), seqops.Rotation(48), 2 ** 31 - 1
    k, v = (torch.randn(1, 1, 48, generator=gen(i), device="cuda").half() for i in (1, 2))
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    cache.store(k.expand(n, 1, 48), v.expand(n, 1, 48), table, seqops.Batch([0], [n], [0]), rotation=rot)
    pos = np.arange(32)
    want, tol = plain.rotate(np.broadcast_to(as64(k), (32, 1, 48)), pos, rot.frequencies, rot.gain, rot.pairs)
    near(torch.cat([cache.k[2, 0], cache.k[0, 0]])[:, None], want, tol, torch.float16)
    assert torch.equal(cache.v[[2, 0], 0], v.expand(2, 16, 48)) and (cache.k[[1, 3]] == 0).all() and (cache.v[[1, 3]] == 0).all()
