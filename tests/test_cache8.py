"""The cache in 8 bits where no GPU is needed: what its calls refuse, before anything is launched."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from atomserve_amd.kernels import ops

BF16, F32, I32, E4M3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def nothing_is_launched(monkeypatch):
    def call(name, *args):
        raise AssertionError(f"{name} would have been launched")

    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(ops, "_addresses", lambda *tensors: [0] * len(tensors))
    monkeypatch.setattr(ops, "_stream8", lambda here: 0)
    monkeypatch.setattr(ops, "_device", lambda: 0)
    monkeypatch.setattr(ops, "_compute_units", 256)
    with FakeTensorMode():  # tensors that say they are on the GPU, without memory
        yield


def tensor(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda:0")


def cache(KV=2, bs=16, D=64, NB=4, **kw):
    made = {"k_pages": tensor(NB, KV, bs, D, dtype=E4M3), "v_pages": tensor(NB, KV, bs // 16, D, 16, dtype=E4M3),
            "k_scales": tensor(NB, KV, bs // 16, dtype=F32), "v_scales": tensor(NB, KV, bs // 16, dtype=F32)}  # fmt: skip
    return {**made, **kw}


def append(T=3, H=4, KV=2, D=64, **kw):
    args = {"qkv": tensor(T, H + 2 * KV, D), "q_weight": None, "k_weight": None, "cos_sin": tensor(T, D // 2, 2, dtype=F32),
            "slots": tensor(T, dtype=I32), "q_out": tensor(T, H, D), **cache(KV, D=D), "num_heads": H, "num_kv_heads": KV, "eps": 1e-6}  # fmt: skip
    ops.qk_norm_rope_store8(**{**args, **kw})


def single(T=3, H=4, KV=2, D=64, **kw):
    args = {"q": tensor(T, H, D), **cache(KV, D=D), "items": None, "positions": tensor(T, dtype=I32), "tok_row": None,
            "block_tables": tensor(T, 4, dtype=I32), "out": tensor(T, H, D), "scale": 0.1, "window": 0, "max_context": 64}  # fmt: skip
    ops.attn_single_query8(**{**args, **kw})


def prompt(T=70, H=4, KV=2, D=64, **kw):
    args = {"q": tensor(T, H, D), **cache(KV, D=D), "tiles": tensor(2, 4, dtype=I32), "block_tables": tensor(1, 8, dtype=I32),
            "out": tensor(T, H, D), "scale": 0.1, "window": 0, "max_context": 70}  # fmt: skip
    ops.attn_prefill8(**{**args, **kw})


def fresh(T=3, H=4, KV=2, D=64, **kw):
    args = {"qkv": tensor(T, H + 2 * KV, D), "q_weight": None, "k_weight": None, "cos_sin": tensor(T, D // 2, 2, dtype=F32),
            "slots": tensor(T, dtype=I32), "eps": 1e-6, "store_kv": True, **cache(KV, D=D), "positions": tensor(T, dtype=I32),
            "block_tables": tensor(T, 4, dtype=I32), "out": tensor(T, H, D), "num_heads": H, "scale": 0.1, "window": 0, "max_context": 64}  # fmt: skip
    ops.attn_decode_fresh8(**{**args, **kw})


@pytest.mark.parametrize("call", [append, single, prompt, fresh])
def test_what_fits_goes_to_the_kernel(call):
    with pytest.raises(AssertionError, match="would have been launched"):
        call()


@pytest.mark.parametrize("call", [append, single, prompt, fresh])
@pytest.mark.parametrize("wrong", [
    {"k_pages": lambda: tensor(4, 2, 16, 64, dtype=BF16)},  # not 8 bits
    {"v_pages": lambda: tensor(4, 2, 64, 16, dtype=E4M3)},  # the layout of a 16-bit cache
    {"v_pages": lambda: tensor(3, 2, 1, 64, 16, dtype=E4M3)},  # fewer pages
    {"k_scales": lambda: tensor(4, 2, 1, dtype=BF16)},
    {"k_scales": lambda: tensor(4, 2, dtype=F32)},
    {"v_scales": lambda: tensor(4, 2, 2, dtype=F32)},
    {"v_scales": lambda: torch.empty(4, 2, 1)},  # on the host
    {"k_pages": lambda: tensor(4, 2, 64, 16, dtype=E4M3).transpose(2, 3)},  # strides
])  # fmt: skip
def test_pages_that_do_not_fit_are_refused(call, wrong):
    with pytest.raises(ops.KernelError):
        call(**{k: v() for k, v in wrong.items()})


@pytest.mark.parametrize("call", [append, single, prompt, fresh])
@pytest.mark.parametrize("D,bs", [(32, 16), (96, 16), (320, 16), (64, 24), (64, 8)])
def test_heads_and_pages_that_no_kernel_takes_are_refused(call, D, bs):
    with pytest.raises(ops.KernelError):
        call(D=D, **cache(D=D, bs=max(16, bs // 16 * 16), k_pages=tensor(4, 2, bs, D, dtype=E4M3)))


@pytest.mark.parametrize("wrong", [
    {"qkv": lambda: tensor(3, 8, 64, dtype=F32)}, {"qkv": lambda: tensor(3, 7, 64)}, {"q_out": lambda: tensor(3, 4, 64, dtype=F32)},
    {"slots": lambda: tensor(4, dtype=I32)}, {"slots": lambda: tensor(3, dtype=torch.int64)}, {"cos_sin": lambda: tensor(3, 34, 2, dtype=F32)},
    {"cos_sin": lambda: tensor(3, 33, 2, dtype=F32)}, {"cos_sin": lambda: tensor(3, 2, 2, dtype=F32)[:, :1].contiguous()},
    {"cos_sin": lambda: tensor(2, 32, 2, dtype=F32)}, {"q_weight": lambda: tensor(64)}, {"k_weight": lambda: tensor(64)},
    {"q_weight": lambda: tensor(64), "k_weight": lambda: tensor(64, dtype=F32)}, {"q_weight": lambda: tensor(32), "k_weight": lambda: tensor(32)},
])  # fmt: skip
def test_appending_refuses(wrong):
    with pytest.raises(ops.KernelError):
        append(**{k: v() for k, v in wrong.items()})


@pytest.mark.parametrize("wrong", [
    {"q": lambda: tensor(3, 4, 64, dtype=F32)}, {"q": lambda: tensor(3, 3, 64), "out": lambda: tensor(3, 3, 64)}, {"out": lambda: tensor(3, 4, 32)},
    {"q": lambda: tensor(3, 4, 128), "out": lambda: tensor(3, 4, 128)}, {"positions": lambda: tensor(2, dtype=I32)},
    {"block_tables": lambda: tensor(2, 4, dtype=I32)}, {"max_context": lambda: 65}, {"window": lambda: -1}, {"softcap": lambda: -1.0},
    {"window": lambda: 5, "chunk": lambda: 5}, {"part_size": lambda: 32}, {"part_size": lambda: 96}, {"part_size": lambda: 0},
    {"sink": lambda: tensor(3, dtype=F32)}, {"scale": lambda: 0.0}, {"items": lambda: tensor(2, dtype=torch.int64)}, {"tok_row": lambda: tensor(2, dtype=I32)},
])  # fmt: skip
def test_single_queries_refuse(wrong):
    with pytest.raises(ops.KernelError):
        single(**{k: v() for k, v in wrong.items()})


@pytest.mark.parametrize("wrong", [
    {"q": lambda: tensor(70, 4, 64, dtype=F32)}, {"q": lambda: tensor(70, 5, 64), "out": lambda: tensor(70, 5, 64)},
    {"tiles": lambda: tensor(2, 3, dtype=I32)}, {"tiles": lambda: tensor(2, 4, dtype=torch.int64)}, {"max_context": lambda: 129},
    {"keep_first": lambda: -1}, {"q": lambda: tensor(70, 4, 128), "out": lambda: tensor(70, 4, 128)},
])  # fmt: skip
def test_prompts_refuse(wrong):
    with pytest.raises(ops.KernelError):
        prompt(**{k: v() for k, v in wrong.items()})


@pytest.mark.parametrize("wrong", [
    {"qkv": lambda: tensor(3, 8, 64, dtype=F32)}, {"qkv": lambda: tensor(3, 9, 64)}, {"num_heads": lambda: 3}, {"out": lambda: tensor(3, 4, 64, dtype=F32)},
    {"slots": lambda: tensor(2, dtype=I32)}, {"cos_sin": lambda: tensor(3, 34, 2, dtype=F32)}, {"cos_sin": lambda: tensor(2, 32, 2, dtype=F32)},
    {"q_weight": lambda: tensor(64)}, {"positions": lambda: tensor(4, dtype=I32)}, {"order": lambda: tensor(2, dtype=I32)},
    {"block_tables": lambda: tensor(2, 4, dtype=I32)}, {"max_context": lambda: 65}, {"window": lambda: -1}, {"scale": lambda: 0.0},
    {"scale": lambda: -1.0}, {"part_size": lambda: 32},
    {"qkv": lambda: tensor(3, 8, 256), "k_pages": lambda: tensor(4, 2, 16, 256, dtype=E4M3), "v_pages": lambda: tensor(4, 2, 1, 256, 16, dtype=E4M3),
     "out": lambda: tensor(3, 4, 256), "cos_sin": lambda: tensor(3, 128, 2, dtype=F32)},  # two kernels are faster
    {"qkv": lambda: tensor(3, 34 + 4, 64), "num_heads": lambda: 34, "out": lambda: tensor(3, 34, 64)},  # 17 heads to a kv head
])  # fmt: skip
def test_decode_steps_from_the_projection_refuse(wrong):
    with pytest.raises(ops.KernelError):
        fresh(**{k: v() for k, v in wrong.items()})


@pytest.mark.parametrize("call,name", [(append, "qkv"), (append, "k_scales"), (single, "block_tables"), (prompt, "tiles"), (fresh, "slots")])
def test_tensors_on_another_device_are_refused(monkeypatch, call, name):
    """The kernel goes on the current device's stream."""
    with pytest.raises(AssertionError, match="would have been launched") as launched:
        call()
    del launched
    monkeypatch.setattr(ops, "_device", lambda: 1)
    with pytest.raises(ops.KernelError, match="current device is cuda:1"):
        call()
    monkeypatch.setattr(ops, "_device", lambda: 0)
    shapes = {"qkv": (3, 8, 64), "k_scales": (4, 2, 1), "block_tables": (3, 4), "tiles": (2, 4), "slots": (3,)}
    dtype = {"qkv": BF16, "k_scales": F32}.get(name, I32)
    with pytest.raises(ops.KernelError, match=f"{name} lies on cuda:1"):
        call(**{name: torch.empty(shapes[name], dtype=dtype, device="cuda:1")})


def test_nothing_to_do_launches_nothing():
    single(items=tensor(0, dtype=I32))
    prompt(tiles=tensor(0, 4, dtype=I32))
    fresh(T=0)


def test_which_heads_the_cache_takes():
    takes = ops.cache8_supported
    assert takes(BF16, 32, 8, 128, 16, 128) and takes(BF16, 24, 1, 256, 48, 0) and takes(BF16, 28, 4, 64, 64, 8)
    assert not takes(F32, 32, 8, 128, 16) and not takes(BF16, 32, 8, 96, 16) and not takes(BF16, 32, 8, 128, 8) and not takes(BF16, 9, 2, 128, 16)
    assert not takes(BF16, 32, 8, 128, 16, 12) and not takes(BF16, 8, 8, 320, 16)
    assert [ops._share8(g) for g in (1, 7, 16, 17, 24, 32, 40)] == [1, 1, 1, 17, 2, 2, 4]


# ---- pools and the models that ask for them -----------------------------------------------------------


def real(fn):
    """Runs with real tensors on the host."""
    from torch.utils._python_dispatch import _disable_current_modes

    def wrapped(*args, **kw):
        with _disable_current_modes():
            return fn(*args, **kw)

    wrapped.__name__ = fn.__name__
    return wrapped


@real
def test_pools_in_8_bits():
    from atomserve_amd.cache import CacheManager, CachePools
    from atomserve_amd.parts.base import PagedCacheRequest

    requests = {0: PagedCacheRequest(2, 64, bits=8), 1: PagedCacheRequest(2, 64), 2: PagedCacheRequest(2, 64, bits=8)}
    manager = CacheManager(requests, 32, 5, 2)
    assert [g.cache_ids for g in manager.paged_groups] == [[0, 2], [1]]
    pools = CachePools(manager, BF16, "cpu")
    _, k, v = pools.pages(2)
    ks, vs = pools.scales_of(2)
    assert k.dtype == v.dtype == E4M3 and k.shape == (5, 2, 32, 64) and v.shape == (5, 2, 2, 64, 16) and k.is_contiguous() and v.is_contiguous()
    assert ks.shape == vs.shape == (5, 2, 2) and ks.dtype == F32 and not ks.any() and not k.view(torch.uint8).any()
    _, k, v = pools.pages(1)
    assert k.dtype == BF16 and v.shape == (5, 2, 64, 32) and pools.scales_of(1) == (None, None)
    held = sum(t.numel() * t.element_size() for t in [*pools.paged, *(s for s in pools.scales if s is not None)])
    assert held == 5 * CachePools.bytes_per_block(requests, 32, BF16)
    for bad, pages in ((PagedCacheRequest(2, 64, bits=8), 24), (PagedCacheRequest(2, 64, bits=4), 16)):
        with pytest.raises(ValueError):
            CachePools(CacheManager({0: bad}, pages, 5, 2), BF16, "cpu")


@real
def test_which_models_keep_8_bits():
    from atomserve_amd.config.registry import architecture_for
    from atomserve_amd.models.decoder import DecoderModel
    from tests.conftest import TINY_A
    from tests.mumizen_cases import CASES

    def model(raw, dtype=BF16, bits=8):
        arch = architecture_for(raw)
        return DecoderModel(arch.build_plan(arch.parse_config(raw)), dtype, "cpu", cache_bits=bits)

    wide = {**TINY_A, "head_dim": 64}
    assert {r.bits for r in model(wide).cache_requests().values()} == {8}
    assert {r.bits for r in model(wide, bits=0).cache_requests().values()} == {0}
    for raw, dtype in ((TINY_A, BF16), (wide, F32)):  # heads of 16; 32-bit heads
        with pytest.raises(ValueError, match="bfloat16 heads of 64"):
            model(raw, dtype)
    with pytest.raises(ValueError, match="no layer"):
        model(CASES["latent_first"])
    with pytest.raises(ValueError, match="8 bits, not 4"):
        model(wide, bits=4)


def test_the_command_line_names_the_cache():
    from atomserve_amd.engine.cli import build_parser

    assert build_parser().parse_args(["m"]).cache_bits == 0 and build_parser().parse_args(["m", "--cache-bits", "8"]).cache_bits == 8
    with pytest.raises(SystemExit):
        build_parser().parse_args(["m", "--cache-bits", "4"])


# ---- how work is cut ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("KV,group", [(1, 1), (8, 4), (4, 24), (3, 7)])
def test_partitions_cover_what_is_seen(D, KV, group):
    share = ops._share8(group)
    assert group % share == 0 and group // share <= 16 and all(group % n or group // n > 16 for n in range(1, share))
    H = KV * group
    for N in (1, 2, 9, 64, 500):
        for context in (1, 63, 64, 65, 1000, 33_333, 1_000_000):
            for window, keep in ((0, 0), (1, 0), (200, 0), (200, 70), (5000, 1)):
                part, P, workspace = ops._partitions8(N, H, KV * share, D, context, window, None, "cuda:0", keep)
                # no query walks more steps of 64 keys than this: all of them, or those that hold kept keys and those that the window reaches into
                steps = -(-context // 64) if not window else min(-(-context // 64), -(-keep // 64) + (window - 1 + 63) // 64 + 1)
                assert part % 64 == 0 and P * (part // 64) >= steps and 1 <= P <= 65535
                assert (P == 1) == (workspace is None) and (P == 1 or workspace.numel() == N * H * P * (D + 2))
                if N * KV * share >= 384:
                    assert P == 1
                assert ops.contexts_cut8(N, H, KV, D, context, window, keep) == (P > 1)


def test_a_step_whose_queries_see_nothing_is_a_step():
    assert ops._partitions8(3, 32, 8, 128, 0, 0, None, "cuda:0") == (64, 1, None)
    for call in (single, fresh, prompt):
        with pytest.raises(AssertionError, match="would have been launched"):
            call(max_context=0)


def test_a_lone_long_context_is_cut_for_the_whole_gpu():
    part, P, _ = ops._partitions8(1, 32, 8, 128, 131_072, 0, None, "cuda:0")
    assert P * 8 >= 256 and part >= 256
    assert ops._partitions8(1, 32, 8, 128, 100, 0, None, "cuda:0")[1] == 1
    with pytest.raises(ops.KernelError, match="multiples of 64"):
        ops._partitions8(1, 32, 8, 128, 100, 0, 96, "cuda:0")


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("H,KV", [(32, 8), (4, 4), (24, 1)])
def test_pieces_of_a_portion_cover_its_rounds(D, H, KV):
    for tiles in (1, 2, 32, 300):
        for context in (1, 64, 65, 2000, 100_000):
            for window in (0, 100):
                for forced in (None, 1, 3, 100):
                    if context < 64 * (tiles - 1) / 16:
                        continue
                    kind, pieces, rounds = ops._prefill8_plan(tiles, H, KV, D, context, window, None, 0, forced, 256)
                    span = min(context, window + 64) if window else context
                    assert kind in (1, 2) and pieces >= 1
                    if pieces > 1:
                        assert pieces * rounds >= -(-span // 64) and rounds * 64 * pieces < 2 * span + 64 * pieces and (forced is None or pieces <= forced)


def test_a_portion_behind_a_long_prefix_is_cut_and_many_are_not():
    assert ops._prefill8_plan(1, 32, 8, 128, 16_000, 0, None, 0, None, 256)[1] > 1
    assert ops._prefill8_plan(200, 32, 8, 128, 2_000, 0, None, 0, None, 256)[1] == 1
