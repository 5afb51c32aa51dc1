"""An engine whose cache is held in 8 bits: the attention part against a plain form that holds its keys and values in the same 8 bits, and steps of
every kind against each other."""

import math

import pytest
import torch

from atomserve_amd.cache.manager import CacheManager
from atomserve_amd.cache.pools import CachePools
from atomserve_amd.config import EngineConfig
from atomserve_amd.config.registry import architecture_for
from atomserve_amd.engine.batch import Row, StepBatch
from atomserve_amd.engine.engine import create_engine
from atomserve_amd.engine.runner import ModelRunner
from atomserve_amd.engine.sequence import SamplingParams
from atomserve_amd.models.decoder import DecoderModel
from atomserve_amd.parts.base import BuildEnv, build
from atomserve_amd.parts.plan import AttentionSpec, NormSpec, RotarySpec
from atomserve_amd.weights.loader import DictSource, bind_checkpoint
from atomserve_amd.weights.random_init import random_checkpoint
from tests import plain_cache8 as plain8
from tests import plain_kernels as pk

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda:0", torch.bfloat16
RAW = {"architectures": ["Qwen3ForCausalLM"], "vocab_size": 300, "hidden_size": 128, "intermediate_size": 256, "num_hidden_layers": 6,
       "num_attention_heads": 6, "num_key_value_heads": 2, "head_dim": 64, "rms_norm_eps": 1e-6, "rope_theta": 10000.0,
       "tie_word_embeddings": True, "max_position_embeddings": 2048, "hidden_act": "silu"}  # fmt: skip


def make_model(bits=8, std=0.1, **raw):
    arch = architecture_for({**RAW, **raw})
    config = arch.parse_config({**RAW, **raw})
    model = DecoderModel(arch.build_plan(config), BF16, DEV, cache_bits=bits)
    bind_checkpoint(model, arch, config, DictSource(random_checkpoint(arch, config, seed=3, dtype=BF16, device=DEV, std=std)))
    model.env.products.fix()
    return model


@pytest.mark.parametrize("norm,window,bs", [(True, 0, 16), (False, 0, 32), (True, 25, 16)])
def test_attention_part_alone(norm, window, bs):
    """A prompt, then the same request token by token and a portion, against the plain form: projections and roundings to bfloat16 as the part makes
    them, keys and values in the blocks that the part's own cache holds."""
    h, H, KV, D = 96, 6, 2, 64
    spec = AttentionSpec("attention", h, H, KV, D, 1 / math.sqrt(D), NormSpec("rmsnorm", D, 1e-5) if norm else None,
                         RotarySpec("rope_half", D, 5e4), window=window)  # fmt: skip
    mixer = build("mixer", spec, BuildEnv(dtype=BF16, device=torch.device(DEV), cache_bits=8))
    g = torch.Generator(device=DEV).manual_seed(7)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    w = {"qkv.weight": (randn((H + 2 * KV) * D, h) * 0.2).to(BF16), "o.weight": (randn(h, H * D) * 0.1).to(BF16)}
    if norm:
        w |= {"q_norm.weight": (1 + 0.2 * randn(D)).to(BF16), "k_norm.weight": (1 + 0.2 * randn(D)).to(BF16)}
    mixer.bind(w)
    manager = CacheManager({0: mixer.cache_request()}, bs, 16, 2)
    pools = CachePools(manager, BF16, DEV)
    rc, done = manager.new_request(), 0
    for n in (40, 1, 1, 5, 30, 1):
        manager.reserve(rc, done, n)
        batch = StepBatch([Row([0] * n, done, rc.tables, [])], bs, 1, 10, DEV, pools=pools, row_splits=[mixer.row_split()])
        x = randn(n, h).to(BF16)
        got = mixer.forward(x, batch, batch.cache_view(0, True)).double()
        qkv = (x.double() @ w["qkv.weight"].double().T).to(BF16).view(n, H + 2 * KV, D)
        angles = plain8.positions_angles(range(done, done + n), D, 5e4).to(DEV)
        q, k, v = pk.qk_norm_rope(qkv, w.get("q_norm.weight"), w.get("k_norm.weight"), angles, H, KV, 1e-5)
        _, k_pages, v_pages = pools.pages(0)
        cache = (k_pages, v_pages, *pools.scales_of(0))
        table = [max(p, 0) for p in rc.tables[0]]  # pages that a window has given back are seen by nobody
        held_k, held_v = plain8.gathered(cache, table, done + n)
        for held, fresh, scales in ((held_k, k, cache[2]), (held_v, v, cache[3])):  # what was stored is what was projected, to 8 bits
            off = (held[:, done:].transpose(0, 1) - fresh.double()).abs()
            # a projection's last bfloat16 digit may differ (2^-7 of it), a norm carries a row's differences on: 2^-6 of the largest
            assert bool((off <= fresh.abs() * (plain8.HALF_STEP + 2.0**-7) + fresh.abs().amax(-1, keepdim=True) * 2.0**-6).all())
        heads, bound = zip(*[plain8.attend(q[i], held_k[:, : done + i + 1], held_v[:, : done + i + 1], done + i, spec.scale, window) for i in range(n)])
        want = torch.stack(heads).view(n, H * D) @ w["o.weight"].double().T
        # the bfloat16 queries may be a digit off (2^-7 of a score's terms: less than 2^-4 of a weight here), heads and results are rounded
        assert bool(((got - want).abs() <= 2.0**-4 * want.abs().amax()).all()), float((got - want).abs().max() / want.abs().max())
        done += n
        manager.release_behind_window(rc, done)


STEPS = ([("a", 5)], [("b", 14)], [("c", 17)], [("a", 1), ("d", 40)], [("b", 100), ("c", 1), ("a", 3)], [("e", 200)],
         [("a", 1), ("b", 1), ("c", 30), ("e", 90)], [("a", 1), ("b", 1), ("e", 1)], [("d", 9), ("a", 2)])  # fmt: skip


def run_steps(model, steps, bs=16, graphs=True):
    manager = CacheManager(model.cache_requests(), bs, 64, 8)
    runner = ModelRunner(model, manager, use_graphs=graphs)
    gen, held, out = torch.Generator().manual_seed(1), {}, []
    for step in steps:
        rows = []
        for rid, n in step:
            cache, at = held.get(rid) or (manager.new_request(), 0)
            assert manager.reserve(cache, at, n)
            rows.append(Row(torch.randint(300, (n,), generator=gen).tolist(), at, cache.tables, [0, n - 1][: min(n, 2)], cache.state_slot))
            held[rid] = (cache, at + n)
        out.append(runner.step(rows).clone())
    return out, runner.pools


def test_layers_from_a_list_are_the_layers():
    """Prompts, portions beside decoding requests, replayed decode steps: launched from a list and part by part, the same bits."""
    model, other = make_model(), make_model()
    assert model.stretches is not None
    other.stretches = None
    (a, pools_a), (b, pools_b) = run_steps(model, STEPS), run_steps(other, STEPS)
    assert pools_a.paged[0].dtype == torch.float8_e4m3fn and pools_a.scales[0].shape[-1] == 1
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), f"step {i}"
    assert torch.equal(pools_a.paged[0].view(torch.uint8), pools_b.paged[0].view(torch.uint8)) and torch.equal(pools_a.scales[0], pools_b.scales[0])


def test_replayed_decode_steps_are_the_eager_ones():
    """Several replays of the captured steps with other steps between them, rows that pad a bucket among them (they store nothing)."""
    steps = [[("a", 40), ("b", 9), ("c", 70)]] + [[("a", 1), ("b", 1), ("c", 1)]] * 30 + [[("d", 33)]] + [[("d", 1), ("a", 1)]] * 10
    (a, pools_a), (b, pools_b) = run_steps(make_model(), steps), run_steps(make_model(), steps, graphs=False)
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), f"step {i}"
    assert torch.equal(pools_a.paged[0].view(torch.uint8), pools_b.paged[0].view(torch.uint8)) and torch.equal(pools_a.scales[0], pools_b.scales[0])


@pytest.mark.parametrize("bs", [16, 48])
def test_a_prompt_in_portions_and_token_by_token_is_the_prompt(bs):
    """The cache holds the same numbers however a request's tokens came, and so the logits agree to what bfloat16 leaves."""
    ids = 150
    whole, pools = run_steps(make_model(num_hidden_layers=2), [[("a", ids)]], bs)
    for cuts in ([64, 86], [7] * 20 + [10], [149, 1]):
        got, others = run_steps(make_model(num_hidden_layers=2), [[("a", n)] for n in cuts], bs)
        last = whole[-1][-1]
        assert (got[-1][-1] - last).abs().max() <= 3e-2 * max(1.0, float(last.abs().max()))
        # the first layer's blocks: projections of other row counts may differ in a last digit; scales are powers of two and rarely move
        assert (pools.scales[0][0] == others.scales[0][0]).float().mean() > 0.97


def test_an_engine_serves_from_8_bits():
    """Continuous batching with few pages (preemption and pages used again), prefixes shared, greedy: the same tokens whether steps are sent ahead or
    not; and memory is what `bytes_per_block` says."""
    model = make_model(num_hidden_layers=2)
    requests, out = model.cache_requests(), []
    prompts = [[5, 17, 3, 250, 299] * 9, [7] * 19, [1], [5, 17, 3, 250, 299] * 9 + [4, 4]]
    for ahead in (True, False):
        engine = create_engine(model, EngineConfig(block_size=16, num_blocks=14, max_model_len=200, max_num_seqs=4, max_num_batched_tokens=32))
        engine.run_ahead = ahead
        out.append(engine.generate(prompts, SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True)))
        pools = engine.runner.pools
        held = sum(t.numel() for t in pools.paged) + 4 * sum(t.numel() for t in pools.scales)
        assert held == 14 * CachePools.bytes_per_block(requests, 16, BF16)
    assert out[0] == out[1] and all(len(t) == 24 for t in out[0])
