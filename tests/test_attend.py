"""What xds_attend draws, and that it says so where there is no GPU."""
import numpy as np
import pytest
import torch

from kv_offload_proto_amd.xds import xds_attend


@pytest.mark.parametrize("tokens", [1, 4, 64])
def test_trees(tokens):
    parent, mask = xds_attend.draw_tree(np.random.default_rng(3), 5, tokens)
    for b in range(5):
        for t in range(tokens):
            path = xds_attend._path(parent[b], t)
            assert path == sorted(set(path)) and path[-1] == t
            assert int(np.uint64(mask[b, t])) == sum(1 << i for i in path)


@pytest.mark.parametrize("prefill,seq_lens,top_k", [(8, [8, 9, 30], 6), (3, [3, 4], 10), (5, [5], 1)])
def test_selections(prefill, seq_lens, top_k):
    got = xds_attend.draw_selection(np.random.default_rng(4), prefill, seq_lens, top_k)
    for row, n in zip(got, seq_lens):
        real = row[row >= 0]
        assert len(set(real)) == len(real) and (real < n).all()
        assert set(range(max(prefill, n - top_k // 2), n)) <= set(real)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is there")
def test_without_a_gpu(capsys):
    assert xds_attend.main([]) == 1
    assert "[xds][ERROR] no GPU visible" in capsys.readouterr().out
