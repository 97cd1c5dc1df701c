"""Attention over a paged cache by more row tiles than a grid has blocks for."""
import numpy as np
import pytest

from test_gpu_paged import Tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_of_a_million_sequences(gpu, half):
    """8 KV heads of 2^20 - 1 sequences, nearly all without rows, three with row tiles for several blocks."""
    seqs = [(0, 0)] * ((1 << 20) - 1)
    seqs[0], seqs[700_000], seqs[-1] = (3, 170), (5, 1), (20, 129)
    t = Tree(gpu, seqs, 8, 8, 32, 16, half)
    t.check()
    assert np.isfinite(t.out()).all()
