"""Which of the two ways a decode step over a cache in 8 bits goes."""

import pytest
import torch

from atomserve_amd.kernels import ops

# (requests, kv heads, head width, tokens) at which one way was measured to be at least a twentieth faster than the other
ONE = [(1, 8, 128, 100), (8, 8, 128, 500), (64, 8, 128, 100), (64, 8, 128, 2048), (96, 4, 128, 700), (512, 1, 128, 800), (8, 8, 128, 16_000), (96, 8, 64, 700),
       (128, 4, 64, 500), (8, 8, 192, 500), (32, 8, 192, 500), (64, 8, 192, 100), (96, 8, 192, 100), (16, 8, 192, 8000), (128, 1, 192, 2048), (32, 4, 192, 2048)]
TWO = [(256, 8, 128, 300), (384, 8, 128, 100), (384, 8, 128, 500), (512, 8, 128, 300), (512, 4, 128, 300), (512, 4, 64, 300), (512, 8, 64, 300), (48, 8, 192, 2048),
       (64, 8, 192, 4000), (40, 8, 192, 3000), (128, 8, 192, 2048), (256, 8, 192, 100), (256, 8, 192, 500), (64, 4, 192, 4000), (384, 4, 192, 500)]  # fmt: skip


@pytest.mark.parametrize("case", ONE)
def test_one_kernel_where_it_is_faster(case):
    assert ops.decode_fresh8_faster(*case)


@pytest.mark.parametrize("case", TWO)
def test_append_and_attention_where_they_are_faster(case):
    assert not ops.decode_fresh8_faster(*case)


@pytest.mark.gpu
def test_both_ways_give_a_server_the_same_logits_and_cache(monkeypatch):
    """Steps of prompts and of single tokens, captured and not, with either way forced."""
    from tests.test_cache8_engine_gpu import make_model, run_steps

    steps = [[("a", 40), ("b", 9), ("c", 70)]] + [[("a", 1), ("b", 1), ("c", 1)]] * 9
    taken = []
    monkeypatch.setattr(ops, "attn_decode_fresh8", lambda *args, real=ops.attn_decode_fresh8, **kw: (taken.append(1), real(*args, **kw)))
    for graphs in (True, False):
        found = []
        for one in (True, False):
            monkeypatch.setattr(ops, "decode_fresh8_faster", lambda *case, one=one: one)
            taken.clear()
            found.append(run_steps(make_model(num_hidden_layers=2), steps, graphs=graphs))
            assert bool(taken) == one
        (a, pools_a), (b, pools_b) = found
        assert all(torch.equal(x, y) for x, y in zip(a, b, strict=True))
        assert torch.equal(pools_a.paged[0].view(torch.uint8), pools_b.paged[0].view(torch.uint8)) and torch.equal(pools_a.scales[0], pools_b.scales[0])
