"""The bounded waits of chunk attention, made to run out in the harmless form: a test knob lets the warp that hands
out the work of the first CTA wait, before it has handed out or loaded anything, for something that
never comes.  After two seconds that wait and those of the CTA's other warps give up, the kernel ends, the word
for it is set and the context stays usable."""
import pytest

from test_gpu_chunk_attention import make, run

pytestmark = pytest.mark.gpu


@pytest.fixture
def stall():
    import kvx_b200
    kvx_b200.lib().kvx_attention_device_error(1)
    yield lambda on: kvx_b200.set_option("chunk_test_stall", int(on))
    kvx_b200.set_option("chunk_test_stall", 0)
    kvx_b200.lib().kvx_attention_device_error(1)


@pytest.mark.parametrize("dim,layout,cache", [(128, "nhd", "same"), (256, "hnd", "same"), (128, "nhd", "f8"), (64, "packed", "same")])
def test_a_wait_that_runs_out(stall, dim, layout, cache):
    """By every way into shared memory, with one stream and with two."""
    import torch
    import kvx_b200
    L = kvx_b200.lib()
    # contexts too short to be cut: every tile is one CTA's
    c = make(dim=dim, layout=layout, cache=cache, lens=((9, 200),) * 200, seed=60)
    clean = run(c, 0.1, max_seq_len=256)
    out = torch.full_like(clean, 7.0)
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    stall(True)
    a.record()
    run(c, 0.1, max_seq_len=256, out=out)
    b.record()
    torch.cuda.synchronize()
    stall(False)
    assert L.kvx_attention_device_error(0) == 1  # read without clearing
    assert L.kvx_attention_device_error(1) == 1  # read and clear
    assert L.kvx_attention_device_error(0) == 0
    left = (out == 7.0).all(-1)
    rest = torch.equal(out[~left], clean[~left])
    assert rest and 0 < int(left.sum()) < left.numel() // 20
    assert 1000 < a.elapsed_time(b) < 4000
    again = run(c, 0.1, max_seq_len=256)
    torch.cuda.synchronize()
    same = torch.equal(again, clean)
    assert same and L.kvx_attention_device_error(0) == 0
