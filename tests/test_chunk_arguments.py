"""Arguments of chunk attention that are refused before the library is called (no GPU needed)."""
import pytest


@pytest.mark.parametrize("limit", [0, -1, -(2 ** 40)])
def test_a_context_limit_without_tokens_is_refused(limit):
    """Not taken for "no limit", which would attend to tokens that the caller excluded."""
    import torch
    from kvx_b200 import ops
    q = torch.zeros((4, 8, 64), dtype=torch.bfloat16)
    cache = torch.zeros((2, 16, 8, 64), dtype=torch.bfloat16)
    table, lens, at = (torch.zeros(s, dtype=torch.int32) for s in ((1, 1), (1,), (2,)))
    with pytest.raises(ValueError, match="max_seq_len"):
        ops.paged_attention_chunk(q, cache, cache, table, lens, at, 0.1, max_seq_len=limit)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nhd", "packed"])
def test_the_same_on_the_gpu(layout):
    from test_gpu_chunk_attention import make, run
    c = make(lens=((5, 40),), layout=layout)
    with pytest.raises(ValueError, match="max_seq_len"):
        run(c, 0.1, max_seq_len=0)
    run(c, 0.1, max_seq_len=1)
