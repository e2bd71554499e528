"""Which blocks a group behind a shared prefix takes on this device (chk_attn_prefix_q4), and what
they give: 33 to 64 (row, head) pairs of a kv head, fewer than a block of many holds."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_attn_views import prefix_cut
from tests.test_gpu_kv4 import KINDS
from tests.test_gpu_views import call, grouped

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,heads,seqs,hd", [("f32", 3, 11, 128), ("f32", 7, 9, 128), ("bf16", 3, 11, 128), ("bf16", 5, 8, 128),
                                                ("f16", 3, 16, 256)])
def test_few_pairs_in_blocks_of_many(have_gpu, kind, heads, seqs, hd):
    """16 kv heads, 33 to 63 pairs: blocks of 16 up to eight tiles of theirs a workgroup of the device,
    one of 64 or 128 behind a prefix that is a tile longer."""
    import torch

    groups = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    nkv, pairs = 16, heads * seqs
    few = -(-pairs // 16)
    limit = 8 * groups // nkv // few  # tiles of the prefix
    for tiles, block in ((limit, 16), (limit + 1, 128 if hd == 128 and kind == "bf16" else 64)):
        tail = ([1, 30, 2, 9, 70, 5, 66, 3] * 2)[:seqs]
        cache, lens, first, shared = grouped(np.random.default_rng(pairs), 64, nkv, hd, [(64 * tiles, tail)], [])
        walks, _ = prefix_cut(heads * nkv, nkv, hd, KINDS[kind], groups, lens, np.arange(seqs + 1), seqs, cache[1].shape[1] * 64,
                              first, shared)
        assert walks[0][[1, 2, 5]].tolist() == [seqs, 64 * tiles, block]
    call(3, (heads * nkv, nkv, hd), 64, lens, [1] * seqs, kind, False, cache=cache, share=(first, shared))
