"""The calls over a cache in 8 bits as programs use them: captured and replayed, on streams of their own, in pools beyond 32 bits, with inputs that are
not finite or start anywhere."""

import pytest
import torch

from tests import plain_cache8 as plain

pytestmark = pytest.mark.gpu
BF16, F32, I32, DEV = torch.bfloat16, torch.float32, torch.int32, "cuda"


@pytest.fixture(scope="module")
def ops():
    from atomserve_amd.kernels import ops

    return ops


def i32(values):
    return torch.tensor(values, dtype=I32, device=DEV)


class Step:
    """What a layer of a mixed step does: two portions of prompts, six single tokens behind contexts that are cut into partitions and, with `fresh`, the same
    tokens' next step from the projection.  All tensors are there once, so that a graph can hold the calls."""

    def __init__(self, ops, seed=0, H=8, KV=2, D=128, bs=32, page0=0, pages=None):
        self.ops, self.H, self.KV, self.D, self.bs = ops, H, KV, D, bs
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.g = g
        need = 100
        self.cache = plain.empty(pages or need + page0, KV, bs, D, DEV)
        part = plain.empty(need, KV, bs, D, DEV)
        plain.fill(part, *(torch.randn(need, KV, bs, D, generator=g, device=DEV) for _ in range(2)))
        for whole, piece in zip(self.cache, part):
            (whole.view(torch.uint8) if whole.element_size() == 1 else whole)[page0 : page0 + need] = piece.view(torch.uint8) if piece.element_size() == 1 else piece
        self.page0, self.need = page0, need
        order = [page0 + p for p in torch.randperm(need, generator=torch.Generator().manual_seed(seed)).tolist()]
        width = 20
        self.contexts = [1, 17, 100, 250, 333, 600]
        self.prompts = [(70, 0), (90, 500)]  # tokens, behind
        tables, at, slots, positions, tiles = [], 0, [], [], []
        for n in self.contexts:
            pages_of = order[at : at + width]
            at += -(-(n + 1) // bs)
            tables.append(pages_of)
            slots.append(pages_of[(n - 1) // bs] * bs + (n - 1) % bs)
            positions.append(n - 1)
        for row, (n, behind) in enumerate(self.prompts, len(tables)):
            pages_of = order[at : at + width]
            at += -(-(n + behind) // bs)
            tables.append(pages_of)
            for i in range(0, n, 64):
                tiles.append((len(slots), min(64, n - i), row, behind + i))
                slots += [pages_of[p // bs] * bs + p % bs for p in range(behind + i, behind + min(i + 64, n))]
                positions += range(behind + i, behind + min(i + 64, n))
        assert at <= need
        T, N = len(slots), len(self.contexts)
        self.T, self.N = T, N
        self.slots, self.positions, self.tiles, self.tables = i32(slots), i32(positions), i32(tiles), i32(tables)
        self.items = i32(range(N))
        self.next_positions = i32(self.contexts)
        self.next_slots = i32([t[n // bs] * bs + n % bs for t, n in zip(tables, self.contexts)])
        self.cos_sin = plain.positions_angles(positions, D).to(DEV)
        self.next_cos_sin = plain.positions_angles(self.contexts, D).to(DEV)
        self.gains = [(1 + 0.3 * torch.randn(D, generator=g, device=DEV)) for _ in range(2)]
        self.qkv = torch.empty(T, H + 2 * KV, D, dtype=BF16, device=DEV)
        self.next_qkv = torch.empty(N, H + 2 * KV, D, dtype=BF16, device=DEV)
        self.q = torch.empty(T, H, D, dtype=BF16, device=DEV)
        self.out = torch.empty(T, H, D, dtype=BF16, device=DEV)
        self.next_out = torch.empty(N, H, D, dtype=BF16, device=DEV)
        self.part = None
        self.new_inputs(seed)

    def new_inputs(self, seed):
        g = torch.Generator(device=DEV).manual_seed(1000 + seed)
        for x in (self.qkv, self.next_qkv):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))

    def calls(self):
        """All of it, on the current stream."""
        ops, scale = self.ops, plain.default_scale(self.D)
        ops.qk_norm_rope_store8(self.qkv, *self.gains, self.cos_sin, self.slots, self.q, *self.cache, self.H, self.KV, 1e-6)
        ops.attn_single_query8(self.q, *self.cache, self.items, self.positions, None if self.tables.shape[0] >= self.T else self.rows(), self.tables, self.out,
                               scale, 0, 600, part_size=128)  # fmt: skip
        ops.attn_prefill8(self.q, *self.cache, self.tiles, self.tables, self.out, scale, 0, 590)
        ops.attn_decode_fresh8(self.next_qkv, *self.gains, self.next_cos_sin, self.next_slots, 1e-6, True, *self.cache, self.next_positions, self.tables,
                               self.next_out, self.H, scale, 0, 601, part_size=64)  # fmt: skip

    def rows(self):
        if self.part is None:  # rows of the tables that tokens read: those of single tokens are asked for
            self.part = torch.zeros(self.T, dtype=I32, device=DEV)
            self.part[: self.N] = self.items
        return self.part

    def state(self):
        held = [c[self.page0 : self.page0 + self.need].clone() for c in (*(x.view(torch.uint8) for x in self.cache[:2]), *self.cache[2:])]
        return [self.out.clone(), self.next_out.clone(), self.q.clone(), *held]

    def put_back(self, held):
        for c, h in zip((*(x.view(torch.uint8) for x in self.cache[:2]), *self.cache[2:]), held):
            c[self.page0 : self.page0 + self.need] = h


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


def forced_pieces(ops, monkeypatch, n=3):
    monkeypatch.setattr(ops, "PREFILL_PIECES", n)


def test_the_step_is_right(ops, monkeypatch):
    """Against 64 bits, before the tests below compare it with itself."""
    forced_pieces(ops, monkeypatch)
    s = Step(ops)
    s.calls()
    scale = plain.default_scale(s.D)
    for t in range(s.T):
        row = t if t < s.N else next(r for f, n, r, _ in s.tiles.tolist() if f <= t < f + n)
        if t >= s.N and t % 13:
            continue
        p = int(s.positions[t])
        if t >= s.N:  # the single tokens' blocks have grown by the next step's tokens since
            k, v = plain.gathered(s.cache, s.tables[row].tolist(), p + 1)
            want, bound = plain.attend(s.q[t], k, v, p, scale)
            assert bool(((s.out[t].double() - want).abs() <= bound).all()), t
    q = torch.empty(s.N, s.H, s.D, dtype=BF16, device=DEV)
    ops.qk_norm_rope_store8(s.next_qkv, *s.gains, s.next_cos_sin, None, q, None, None, None, None, s.H, s.KV, 1e-6, store_kv=False)
    for t in range(s.N):
        p = int(s.next_positions[t])
        k, v = plain.gathered(s.cache, s.tables[t].tolist(), p + 1)
        want, bound = plain.attend(q[t], k, v, p, scale)
        assert bool(((s.next_out[t].double() - want).abs() <= bound).all()), t


def test_captured_and_replayed_beside_another_graph(ops, monkeypatch):
    """Two graphs of the same calls on other data, replayed in turn with eager work between: every replay gives what the eager calls give, for new inputs."""
    forced_pieces(ops, monkeypatch)
    steps, graphs, starts = [Step(ops, 0), Step(ops, 5, H=16, KV=4, D=64, bs=48)], [], []
    for s in steps:
        s.calls()  # libraries and attributes are loaded before a capture
        torch.cuda.synchronize()
        starts.append(s.state()[3:])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.calls()
        graphs.append(graph)
    for seed in range(4):
        wanted = []
        for s, start in zip(steps, starts):
            s.new_inputs(seed)
            s.put_back(start)
            s.calls()
            wanted.append(s.state())
            s.put_back(start)
            s.out.fill_(3.0)
            s.next_out.fill_(3.0)
        order = (0, 1) if seed % 2 else (1, 0)
        for i in order:
            graphs[i].replay()
        filler = torch.randn(1 << 20, device=DEV).sort()[0]  # eager work whose memory may be what a workspace was
        torch.cuda.synchronize()
        assert filler.numel() and all(same(s.state(), w) for s, w in zip(steps, wanted)), seed


def test_two_streams_at_once(ops, monkeypatch):
    """The calls on two streams of their own at the same time, several times over: the results of the calls one after the other."""
    forced_pieces(ops, monkeypatch)
    steps = [Step(ops, 1), Step(ops, 2)]
    starts = [s.state()[3:] for s in steps]
    wanted = []
    for s, start in zip(steps, starts):
        s.calls()
        wanted.append(s.state())
        s.put_back(start)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.calls()
        torch.cuda.synchronize()
        for s, w, start in zip(steps, wanted, starts):
            assert same(s.state(), w)
            s.put_back(start)
        torch.cuda.synchronize()


def test_pools_beyond_32_bits(ops, monkeypatch):
    """Pages whose bytes lie behind the first 2^32 of a pool: the results and bytes of the same pages at its start."""
    forced_pieces(ops, monkeypatch)
    near = Step(ops, 3, H=8, KV=4, D=128, bs=32)
    page_bytes = near.KV * near.bs * near.D
    far_page = (1 << 32) // page_bytes + 5
    far = Step(ops, 3, H=8, KV=4, D=128, bs=32, page0=far_page)
    assert far.cache[0].numel() > 1 << 32
    for s in (near, far):
        s.calls()
    assert same(near.state(), far.state())
    assert not bool(far.cache[2][:far_page].any()) and not bool(far.cache[0].view(torch.uint8)[: near.need].any())


@pytest.mark.parametrize("kw", [{}, {"softcap": 8.0}, {"sink": True}], ids=str)
@pytest.mark.parametrize("part", [64, 4096])
def test_a_query_that_is_not_finite_is_nan_and_its_neighbours_are_not(ops, monkeypatch, kw, part):
    H, KV, D, bs, L = 4, 2, 128, 16, 200
    g = torch.Generator(device=DEV).manual_seed(0)
    cache = plain.empty(16, KV, bs, D, DEV)
    plain.fill(cache, *(torch.randn(16, KV, bs, D, generator=g, device=DEV) for _ in range(2)))
    q = torch.randn(L, H, D, generator=g, device=DEV).to(BF16)
    bad = q.clone()
    bad[3, 1, 7], bad[100, 2, 64], bad[199, 3, 0] = float("nan"), float("inf"), -float("inf")
    hit = torch.zeros(L, H, dtype=torch.bool, device=DEV)
    hit[3, 1] = hit[100, 2] = hit[199, 3] = True
    tables, positions = i32([list(range(13))]), i32(range(L))
    tiles = i32([(i, min(64, L - i), 0, i) for i in range(0, L, 64)])
    for pieces in (1, 2):
        monkeypatch.setattr(ops, "PREFILL_PIECES", pieces)
        for call in (
            lambda x, out: ops.attn_single_query8(x, *cache, None, positions, torch.zeros(L, dtype=I32, device=DEV), tables, out, 0.1, 0, L, part_size=part, **kw),
            lambda x, out: ops.attn_prefill8(x, *cache, tiles, tables, out, 0.1, 0, L, **kw),
        ):  # fmt: skip
            clean, got = torch.empty_like(q), torch.empty_like(q)
            call(q, clean)
            call(bad, got)
            assert bool(got[hit].isnan().all()) and bool(clean.isfinite().all())
            assert torch.equal(got[~hit], clean[~hit])


def test_tensors_that_do_not_start_on_16_bytes_are_refused(ops):
    from atomserve_amd.kernels.ops import KernelError

    s = Step(ops)
    odd = lambda x: torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)  # noqa: E731
    scale = plain.default_scale(s.D)
    with pytest.raises(KernelError):
        ops.qk_norm_rope_store8(odd(s.qkv), *s.gains, s.cos_sin, s.slots, s.q, *s.cache, s.H, s.KV, 1e-6)
    with pytest.raises(KernelError):
        ops.qk_norm_rope_store8(s.qkv, *s.gains, odd(s.cos_sin), s.slots, s.q, *s.cache, s.H, s.KV, 1e-6)
    with pytest.raises(KernelError):
        ops.attn_single_query8(odd(s.q), *s.cache, s.items, s.positions, s.rows(), s.tables, s.out, scale, 0, 600)
    with pytest.raises(KernelError):
        ops.attn_prefill8(s.q, *s.cache, s.tiles, s.tables, odd(s.out), scale, 0, 590)
    with pytest.raises(KernelError):
        ops.attn_decode_fresh8(odd(s.next_qkv), *s.gains, s.next_cos_sin, s.next_slots, 1e-6, True, *s.cache, s.next_positions, s.tables, s.next_out, s.H,
                               scale, 0, 601)  # fmt: skip


@pytest.mark.parametrize("bs", [256, 1040])
def test_large_pages(ops, bs):
    from tests.test_cache8_gpu import prompt, single

    single(ops, 8, 2, 128, bs, [1, 255, 256, 257, 1039, 1040, 1041, 1500])
    single(ops, 7, 1, 64, bs, [2500, 3], part_size=128, window=1100)
    prompt(ops, 4, 2, 128, bs, [(70, 0), (33, 1030), (100, 200)])


def test_a_step_whose_queries_see_nothing(ops):
    s = Step(ops)
    none = torch.full((s.N,), -1, dtype=I32, device=DEV)
    before = s.state()[3:]
    for part in (None, 64):
        out = torch.full((s.N, s.H, s.D), 7.0, dtype=BF16, device=DEV)
        ops.attn_single_query8(s.q[: s.N], *s.cache, None, none, None, s.tables, out, 0.1, 0, 0, part_size=part)
        assert not bool(out.any())
        out.fill_(7.0)
        ops.attn_decode_fresh8(s.next_qkv, *s.gains, s.next_cos_sin, none, 1e-6, True, *s.cache, none, s.tables, out, s.H, 0.1, 0, 0, part_size=part)
        assert not bool(out.any()) and same(s.state()[3:], before)


def test_many_tokens(ops):
    """70,001 single queries, and as many tokens of portions, in one call: the results of calls of a thousand."""
    H, KV, D, bs, T = 6, 3, 64, 16, 70_001
    g = torch.Generator(device=DEV).manual_seed(0)
    cache = plain.empty(30, KV, bs, D, DEV)
    plain.fill(cache, *(torch.randn(30, KV, bs, D, generator=g, device=DEV) for _ in range(2)))
    q = torch.randn(T, H, D, generator=g, device=DEV).to(BF16)
    tables = i32([list(range(r, r + 10)) for r in (0, 10, 20)])
    positions, rows = torch.randint(-1, 150, (T,), generator=g, device=DEV, dtype=I32), torch.randint(0, 3, (T,), generator=g, device=DEV, dtype=I32)
    whole, cut = torch.empty_like(q), torch.empty_like(q)
    ops.attn_single_query8(q, *cache, None, positions, rows, tables, whole, 0.125, 0, 150, part_size=192)
    for at in range(0, T, 1000):
        part = slice(at, min(at + 1000, T))
        ops.attn_single_query8(q[part], *cache, None, positions[part], rows[part], tables, cut[part], 0.125, 0, 150, part_size=192)
    assert torch.equal(whole, cut)
    tiles = [(at, min(64, T - at), at % 3, at % 90) for at in range(0, T, 64)]
    ops.attn_prefill8(q, *cache, i32(tiles), tables, whole, 0.125, 0, 154, query_tiles=1)
    for at in range(0, len(tiles), 16):
        ops.attn_prefill8(q, *cache, i32(tiles[at : at + 16]), tables, cut, 0.125, 0, 154, query_tiles=1)
    assert torch.equal(whole, cut)


def test_many_tokens_appended(ops):
    """70,001 tokens in one call, runs and single tokens and some that are not kept: the bytes of calls of a thousand."""
    H, KV, D, bs, T = 2, 3, 64, 16, 70_001
    g = torch.Generator(device=DEV).manual_seed(0)
    qkv = torch.randn(T, H + 2 * KV, D, generator=g, device=DEV).to(BF16)
    cos_sin = torch.randn(T, D // 2, 2, generator=g, device=DEV)
    slots = torch.arange(T, device=DEV, dtype=I32)
    slots[40_000:] = (40_000 // 16 + torch.arange(T - 40_000, device=DEV, dtype=I32)) * 16 + 7  # from here on single tokens, each in a block of its own
    slots[torch.randint(0, T // 16, (500,), generator=g, device=DEV) * 16 + 15] = -1
    one, many = (plain.empty(40_000 // 16 + T - 40_000, KV, bs, D, DEV) for _ in range(2))
    queries = [torch.empty(T, H, D, dtype=BF16, device=DEV) for _ in range(2)]
    ops.qk_norm_rope_store8(qkv, None, None, cos_sin, slots, queries[0], *one, H, KV, 0.0)
    for at in range(0, T, 1008):
        part = slice(at, min(at + 1008, T))
        ops.qk_norm_rope_store8(qkv[part], None, None, cos_sin[part], slots[part], queries[1][part], *many, H, KV, 0.0)
    assert torch.equal(*queries) and all(same([a.view(torch.uint8) if a.element_size() == 1 else a], [b.view(torch.uint8) if b.element_size() == 1 else b])
                                         for a, b in zip(one, many))  # fmt: skip
