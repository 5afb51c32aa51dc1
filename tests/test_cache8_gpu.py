"""The kernels of the cache in 8 bits against plain 64-bit forms (tests/plain_cache8.py), at the sizes and masks where they can go wrong."""

import pytest
import torch

from tests import plain_cache8 as plain
from tests import plain_kernels as pk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, I32, U8, E4M3 = torch.float32, torch.bfloat16, torch.int32, torch.uint8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from atomserve_amd.kernels import ops as module

    return module


def i32(values):
    return torch.tensor(values, dtype=I32, device=DEV)


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(U8), b.contiguous().view(U8))


# ---- appending ------------------------------------------------------------------------------------------


class Appender:
    """A cache and the calls that fill it; `want` holds what every stored token's keys and values were, in 64 bits."""

    def __init__(self, ops, H, KV, D, bs, pages, R=None, norm=F32, seed=0, magnitude=1.0):
        self.ops, self.H, self.KV, self.D, self.bs = ops, H, KV, D, bs
        self.R = D if R is None else R
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.cache = plain.empty(pages, KV, bs, D, DEV)
        self.gains = [None, None]
        if norm is not None:
            self.gains = [(1 + 0.3 * torch.randn(D, generator=self.g, device=DEV)).to(norm) for _ in range(2)]
        self.want_k = torch.zeros(pages, KV, bs, D, dtype=torch.float64, device=DEV)
        self.want_v = torch.zeros_like(self.want_k)
        self.magnitude, self.eps = magnitude, 1e-6

    def put(self, slots, positions, qkv=None, store=True):
        T = len(slots)
        if qkv is None:
            size = torch.exp(torch.randn(T, 1, 1, generator=self.g, device=DEV)) * self.magnitude
            qkv = (torch.randn(T, self.H + 2 * self.KV, self.D, generator=self.g, device=DEV) * size).to(BF16)
        cos_sin = plain.positions_angles(positions, self.R).to(DEV) if self.R else None
        q = torch.full((T, self.H, self.D), 9.0, dtype=BF16, device=DEV)
        self.ops.qk_norm_rope_store8(qkv, *self.gains, cos_sin, i32(slots), q, *self.cache, self.H, self.KV, self.eps, store_kv=store)
        want_q, k, v = (x.double() for x in pk.qk_norm_rope(qkv, *self.gains, cos_sin, self.H, self.KV, self.eps))
        for x in (k, v):
            x[~x.isfinite()] = 0
        off = (q.double() - want_q).abs()
        assert bool((off <= want_q.abs() * 2.0**-8 + 2.0**-18 * want_q.abs().amax(-1, keepdim=True) + 1e-30).all())
        if store:
            for t, slot in enumerate(slots):
                if 0 <= slot < len(self.want_k) * self.bs:
                    self.want_k[slot // self.bs, :, slot % self.bs] = k[t]
                    self.want_v[slot // self.bs, :, slot % self.bs] = v[t]
        return q

    def held(self):
        return plain.keys_of(*self.cache[::2]), plain.values_of(*self.cache[1::2])

    def check(self, slots, roundings=1):
        """Every slot holds its numbers: one rounding (with `roundings` 2: of a block whose scale grew since, whose small numbers were rounded again
        at every growth, by half a smallest step of scales that double at least: two of the last one's in all); 2^-18 for the norm and the turn in 32 bits."""
        slots = torch.tensor(sorted(set(s for s in slots if s >= 0)), device=DEV)
        page, at = slots // self.bs, slots % self.bs
        for got, want, scales, exact in zip(self.held(), (self.want_k, self.want_v), self.cache[2:], (False, True)):
            got, want, s = got[page, :, at], want[page, :, at], scales[page, :, at // 16].double()[..., None]
            slack = 0.0 if exact else 2.0**-18 * want.abs().amax(-1, keepdim=True)
            step = torch.maximum(want.abs() * plain.HALF_STEP, plain.SMALLEST_HALF_STEP * s) + (2 * plain.SMALLEST_HALF_STEP * s if roundings > 1 else 0)
            assert bool(((got - want).abs() <= step + slack).all()), float(((got - want).abs() - step - slack).max())

    def check_scales(self, blocks):
        """blocks: {block of 16 slots: its stored slots}; scales are those of the largest magnitude."""
        for block, slots in blocks.items():
            page, sub = block * 16 // self.bs, block * 16 % self.bs // 16
            at = [s % self.bs for s in slots]
            for want, scales in ((self.want_k, self.cache[2]), (self.want_v, self.cache[3])):
                amax = want[page][:, at].abs().amax((-1, -2)).tolist()
                assert scales[page, :, sub].tolist() == [plain.scale_of(a) for a in amax]


def by_block(slots):
    blocks = {}
    for s in slots:
        blocks.setdefault(s // 16, []).append(s)
    return blocks


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("H,KV,bs,rotary,norm", [(4, 2, 16, 1.0, F32), (5, 1, 48, 0.5, BF16), (3, 3, 32, 0.0, None), (7, 7, 16, 0.125, F32)])
def test_appending_prompts_and_single_tokens(ops, D, H, KV, bs, rotary, norm):
    """Portions that begin and end anywhere in a block, single tokens, tokens that store nothing, in one call; then a second call that goes on in
    the blocks."""
    a = Appender(ops, H, KV, D, bs, 16, R=int(D * rotary), norm=norm)
    first = list(range(0, 37)) + [-1, -1] + [160 + i for i in range(3)] + [240] + [16 * bs + 5, 2**31 - 1] + list(range(96, 112))
    a.put(first, list(range(len(first))))
    mine = [s for s in first if 0 <= s < 16 * bs]
    a.check(mine)
    a.check_scales(by_block(mine))
    second = [37, 38, 163, 241, -1] + list(range(112, 130))
    a.put(second, list(range(1000, 1000 + len(second))))
    a.check(mine + second, 2)
    a.check_scales(by_block(mine + [s for s in second if s >= 0]))


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32)])
def test_a_block_holds_the_same_however_its_tokens_come(ops, D, bs):
    """48 tokens at once, in portions, one by one: the same scales, and the same numbers but where one that fell under the smallest normal was rounded twice."""
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv = torch.randn(48, 6, D, generator=g, device=DEV) * torch.exp(2 * torch.randn(48, 1, 1, generator=g, device=DEV))
    held = []
    for cuts in ([48], [5, 30, 48], list(range(1, 49))):
        a = Appender(ops, 2, 2, D, bs, 4)
        start = 0
        for end in cuts:
            a.put(list(range(start, end)), list(range(start, end)), qkv[start:end].to(BF16))
            start = end
        a.check(range(48), 2)
        held.append(a)
    for other in held[1:]:
        for x, y in zip(held[0].cache[2:], other.cache[2:]):
            assert torch.equal(x, y)
        for x, y, s in zip(held[0].held(), other.held(), other.cache[2:]):
            small = 2.0**-6 * s.double().repeat_interleave(16, 2)[..., None]
            assert bool(((x == y) | (x.abs() <= small)).all())
            assert bool(((x - y).abs() <= 3 * 2.0**-9 * s.double().repeat_interleave(16, 2)[..., None]).all())


def test_a_block_that_starts_again_forgets_and_what_is_not_written_stays(ops):
    a = Appender(ops, 2, 2, 64, 16, 3, magnitude=1e4)
    a.put(range(0, 32), range(32))
    large = [x.clone() for x in a.cache]
    a.magnitude = 1e-3
    a.put([16, 17], [16, 17])  # the second page is another request's now
    assert (a.cache[3][1] < large[3][1]).all()  # keys are normed, values are not
    a.check([16, 17])
    for pages, before in zip(a.cache[:2], large[:2]):
        assert same_bytes(pages[0], before[0]) and same_bytes(pages[2], before[2])
    assert same_bytes(a.cache[0][1, :, 2:], large[0][1, :, 2:]) and same_bytes(a.cache[1][1][..., 2:], large[1][1][..., 2:])
    for scales, before in zip(a.cache[2:], large[2:]):
        assert torch.equal(scales[0], before[0]) and torch.equal(scales[2], before[2])


def test_zeros_extremes_and_numbers_that_are_not_finite(ops):
    a = Appender(ops, 1, 1, 64, 16, 8, R=0, norm=None)
    qkv = torch.zeros(6, 3, 64, device=DEV)
    qkv[1, 1:] = 3.3e38  # beyond 448 * 2^119: kept as that
    qkv[2, 1:] = 1e-38  # under the least scale's smallest number: zero
    qkv[3, 1:, :32] = float("inf")
    qkv[3, 1:, 32:48] = float("nan")
    qkv[3, 1:, 48:] = 2.0
    qkv[4, 1:] = 448.0
    qkv[5, 1:] = 450.0
    slots = [16 * i for i in range(6)]
    a.put(slots, slots, qkv.to(BF16))
    k, v = a.held()
    for x in (k, v):
        assert (x[0, 0, 0] == 0).all() and (x[2, 0, 0] == 0).all() and (x[1, 0, 0] == 448 * 2.0**119).all()
        assert (x[3, 0, 0, :48] == 0).all() and (x[3, 0, 0, 48:] == 2).all() and (x[4, 0, 0] == 448).all() and (x[5, 0, 0] == 448).all()
    for s in a.cache[2:]:
        assert s[:6, 0, 0].tolist() == [2.0**-100, 2.0**119, 2.0**-100, plain.scale_of(2.0), 1.0, 2.0]
    a.put([17], [1], torch.full((1, 3, 64), 5.0, device=DEV).to(BF16))  # goes on behind the extreme: its scale stays
    assert a.cache[3][1, 0, 0] == 2.0**119


def test_queries_alone_store_nothing(ops):
    a = Appender(ops, 5, 2, 128, 16, 2)
    before = [x.clone() for x in a.cache]
    a.put([0, 1, 2], [0, 1, 2], store=False)
    ops.qk_norm_rope_store8(torch.randn(2, 9, 128, device=DEV).to(BF16), None, None, None, None, torch.empty(2, 5, 128, dtype=BF16, device=DEV),
                            None, None, None, None, 5, 2, 0.0, store_kv=False)  # fmt: skip
    assert all(same_bytes(x, y) for x, y in zip(a.cache, before))


# ---- attention ------------------------------------------------------------------------------------------------


def requests(KV, D, bs, lengths, seed=0, spare=3):
    """A full cache and block tables [R, W] of requests of these lengths; every entry behind a request's pages is none of the pool's."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-max(n, 1) // bs) for n in lengths]
    pages = sum(need) + spare
    cache = plain.empty(pages, KV, bs, D, DEV)
    loud = 1 + 6 * (torch.rand(1, 1, 1, D, generator=g, device=DEV) < 0.05)
    size = torch.exp(torch.randn(pages, KV, bs, 1, generator=g, device=DEV))
    plain.fill(cache, torch.randn(pages, KV, bs, D, generator=g, device=DEV) * loud,
               torch.randn(pages, KV, bs, D, generator=g, device=DEV) * size)  # fmt: skip
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at : at + n] + [-1 if at % 2 else 10**9] * (max(need) - n))
        at += n
    return cache, tables, g


def single(ops, H, KV, D, bs, lengths, seed=0, items=None, out_dtype=BF16, tables_of=None, row_of=None, **kw):
    cache, tables, g = requests(KV, D, bs, lengths, seed)
    T = len(lengths)
    q = (torch.randn(T, H, D, generator=g, device=DEV) * 1.5).to(BF16)
    out = torch.full((T, H, D), 7.0, dtype=out_dtype, device=DEV)
    scale = plain.default_scale(D)
    window, part = kw.get("window", 0), kw.pop("part_size", None)
    given = tables if tables_of is None else tables_of(tables)
    ops.attn_single_query8(q, *cache, None if items is None else i32(items), i32([n - 1 for n in lengths]), None if row_of is None else i32(row_of),
                           i32(given), out, scale, window, max(max(lengths), 1), part_size=part,
                           **{k: v for k, v in kw.items() if k != "window"})  # fmt: skip
    sink = kw.get("sink", False)
    sink = sink if isinstance(sink, torch.Tensor) else torch.zeros(H, device=DEV) if sink else None
    for t in range(T) if items is None else items:
        r = t if row_of is None else row_of[t]
        k, v = plain.gathered(cache, tables[r], lengths[t])
        want, bound = plain.attend(q[t], k, v, lengths[t] - 1, scale, window, kw.get("keep_first", 0) if window else 0, kw.get("chunk", 0),
                                   kw.get("softcap", 0.0), sink)  # fmt: skip
        off = (out[t].double() - want).abs()
        assert bool((off <= bound).all()), (t, lengths[t], float((off - bound).max()))
    return out


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 130, 700]


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("H,KV,bs", [(2, 2, 16), (10, 2, 32), (7, 1, 48), (16, 1, 16), (24, 1, 16)])
def test_single_queries(ops, D, H, KV, bs):
    single(ops, H, KV, D, bs, LENGTHS)


@pytest.mark.parametrize("part", [64, 128, 512])
@pytest.mark.parametrize("kw", [{}, {"window": 1}, {"window": 20}, {"window": 300, "keep_first": 5}, {"window": 100, "keep_first": 200}, {"chunk": 33},
                                {"softcap": 5.0}, {"sink": True}, {"sink": "own", "window": 64}, {"out_dtype": F32, "sink": True}], ids=str)  # fmt: skip
def test_single_queries_masks_and_partitions(ops, part, kw):
    kw = dict(kw)
    if kw.get("sink") == "own":
        kw["sink"] = torch.linspace(-3, 9, 8, device=DEV)
    single(ops, 8, 2, 64, 16, LENGTHS + [1999], part_size=part, **kw)
    single(ops, 8, 2, 64, 16, LENGTHS + [1999], part_size=2048, **kw)


def test_single_queries_as_chosen(ops):
    """Partitions as the sizes say, some tokens only, in another order, several of one row; rows that are not named stay."""
    single(ops, 32, 8, 128, 16, [5000, 1, 300])
    single(ops, 32, 8, 128, 16, [700] * 60 + [33] * 7)
    out = single(ops, 16, 8, 128, 32, [900, 20, 61, 450], items=[3, 0], row_of=[0, 1, 2, 3])
    assert (out[1:3] == 7.0).all()
    single(ops, 4, 2, 64, 16, [300, 299, 300, 12], row_of=[0, 0, 2, 3])


def test_a_query_that_sees_nothing_and_pages_that_were_given_back(ops):
    out = single(ops, 4, 2, 64, 16, [0, 5, 0], sink=True)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    assert (single(ops, 4, 2, 64, 16, [0, 300], part_size=64)[0] == 0).all()

    def behind(tables):  # entries that a window of 40 has left behind name no page
        return [[-1 if 16 * (b + 1) <= n - 40 else e for b, e in enumerate(t)] for t, n in zip(tables, [300, 90])]

    single(ops, 4, 2, 64, 16, [300, 90], window=40, tables_of=behind)


def prompt(ops, H, KV, D, bs, rows, seed=0, out_dtype=BF16, order=None, **kw):
    """rows: (tokens, start)."""
    cache, tables, g = requests(KV, D, bs, [n + s for n, s in rows], seed)
    T = sum(n for n, _ in rows)
    q = (torch.randn(T, H, D, generator=g, device=DEV) * 1.5).to(BF16)
    out = torch.full((T + 1, H, D), 7.0, dtype=out_dtype, device=DEV)
    scale, window, tiles, flat = plain.default_scale(D), kw.get("window", 0), [], 0
    for r, (n, s) in enumerate(rows):
        tiles += [(flat + at, min(64, n - at), r, s + at) for at in range(0, n, 64)]
        flat += n
    tiles.sort(key=lambda t: -(t[1] + t[3]))
    if order:
        tiles = order(tiles)
    ops.attn_prefill8(q, *cache, i32(tiles), i32(tables), out[:T], scale, window, max(n + s for n, s in rows),
                      **{k: v for k, v in kw.items() if k != "window"})  # fmt: skip
    assert (out[T] == 7.0).all()
    sink = kw.get("sink", False)
    sink = sink if isinstance(sink, torch.Tensor) else torch.zeros(H, device=DEV) if sink else None
    t = 0
    for r, (n, s) in enumerate(rows):
        k, v = plain.gathered(cache, tables[r], n + s)
        for i in range(n):
            if n <= 70 or i % 37 < 2 or i == n - 1 or i % 64 in (0, 63):
                want, bound = plain.attend(q[t], k[:, : s + i + 1], v[:, : s + i + 1], s + i, scale, window, kw.get("keep_first", 0) if window else 0,
                                           kw.get("chunk", 0), kw.get("softcap", 0.0), sink)  # fmt: skip
                off = (out[t].double() - want).abs()
                assert bool((off <= bound).all()), (r, i, float((off - bound).max()))
            t += 1
    return out


ROWS = [(1, 0), (15, 0), (16, 5), (17, 63), (64, 64), (65, 1), (130, 0), (33, 400)]


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("H,KV,bs", [(2, 2, 16), (10, 2, 32), (7, 1, 48), (24, 1, 16)])
def test_prompts(ops, D, H, KV, bs):
    prompt(ops, H, KV, D, bs, ROWS)


@pytest.mark.parametrize("kw", [{"window": 1}, {"window": 20}, {"window": 100, "keep_first": 5}, {"window": 64, "keep_first": 200}, {"chunk": 33},
                                {"softcap": 5.0}, {"sink": True}, {"sink": "own", "window": 64}, {"out_dtype": F32}], ids=str)  # fmt: skip
def test_prompts_masks(ops, kw):
    kw = dict(kw)
    if kw.get("sink") == "own":
        kw["sink"] = torch.linspace(-3, 9, 8, device=DEV)
    prompt(ops, 8, 2, 64, 16, ROWS + [(300, 900)], **kw)
    prompt(ops, 8, 2, 128, 16, [(70, 130), (9, 3)], **kw)


@pytest.mark.parametrize("query_tiles", [1, 2])
@pytest.mark.parametrize("pieces", [1, 2, 5])
@pytest.mark.parametrize("kw", [{}, {"window": 300, "keep_first": 70}, {"sink": True, "softcap": 9.0}, {"chunk": 200, "out_dtype": F32}], ids=str)
def test_prompts_cut_along_their_keys(ops, monkeypatch, query_tiles, pieces, kw):
    """Items of every length in a step that is cut: the short ones stay whole."""
    monkeypatch.setattr(ops, "PREFILL_PIECES", pieces)
    ops._prefill8_plan.cache_clear()
    prompt(ops, 6, 2, 64, 32, [(100, 1500), (70, 0), (5, 700), (64, 192)], query_tiles=query_tiles, **kw)
    prompt(ops, 10, 2, 128, 16, [(65, 1100), (40, 20)], query_tiles=query_tiles, **kw)
    ops._prefill8_plan.cache_clear()


def test_prompts_longer(ops):
    prompt(ops, 16, 8, 128, 16, [(500, 0), (200, 3000)])
    prompt(ops, 32, 8, 128, 16, [(64, 6000)])
    prompt(ops, 4, 1, 256, 64, [(129, 1500)])


def test_one_run_of_them_together(ops):
    """A request's prompt in two portions, then tokens one by one beside another request: append and attend, every step against 64 bits of what
    the cache holds."""
    H, KV, D, bs = 8, 2, 128, 16
    a = Appender(ops, H, KV, D, bs, 24, norm=BF16)
    scale, order = plain.default_scale(D), torch.randperm(24, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [order[:12], order[12:]]
    slots = lambda r, p: tables[r][p // bs] * bs + p % bs  # noqa: E731
    done = [0, 0]

    def check(r, p, q, got):
        k, v = plain.gathered(a.cache, tables[r], p + 1)
        want, bound = plain.attend(q, k, v, p, scale)
        assert bool(((got.double() - want).abs() <= bound).all())

    for r, n in ((0, 70), (1, 9), (0, 50), (1, 100)):
        at = list(range(done[r], done[r] + n))
        q = a.put([slots(r, p) for p in at], at)
        out = torch.empty_like(q)
        tiles = [(i, min(64, n - i), r, done[r] + i) for i in range(0, n, 64)]
        ops.attn_prefill8(q, *a.cache, i32(tiles), i32(tables), out, scale, 0, done[r] + n)
        done[r] += n
        for i in (0, n // 2, n - 1):
            check(r, at[i], q[i], out[i])
    for _ in range(20):
        q = a.put([slots(r, done[r]) for r in (0, 1)], done)
        out = torch.empty_like(q)
        ops.attn_single_query8(q, *a.cache, None, i32(done), None, i32(tables), out, scale, 0, max(done) + 1)
        for r in (0, 1):
            check(r, done[r], q[r], out[r])
        done = [n + 1 for n in done]
    a.check([slots(r, p) for r in (0, 1) for p in range(done[r])], 2)


@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("H,KV,bs,rotary,norm", [(4, 2, 16, 1.0, F32), (16, 1, 48, 0.5, BF16), (21, 3, 32, 0.0, None)])
@pytest.mark.parametrize("part,window", [(None, 0), (64, 0), (2048, 0), (128, 70)])
def test_a_decode_step_from_the_projection_is_append_and_attention(ops, D, H, KV, bs, rotary, norm, part, window):
    """Bit for bit, results and cache: blocks that are new, go on, or whose scale grows; a token that is not kept; one that the pages hold already; one that sees
    nothing."""
    lengths = [1, 2, 16, 17, 33, 64, 65, 100, 300, 0]
    cache, tables, g = requests(KV, D, bs, lengths)
    T = len(lengths)
    for scales in cache[2:]:  # of earlier tokens: some far smaller than what comes, so that blocks are rewritten
        scales.mul_(torch.exp2(torch.randint(-9, 4, scales.shape, generator=g, device=DEV).float()))
    qkv = (torch.randn(T, H + 2 * KV, D, generator=g, device=DEV) * torch.exp(torch.randn(T, 1, 1, generator=g, device=DEV))).to(BF16)
    gains = [None, None] if norm is None else [(1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(norm) for _ in range(2)]
    R = int(D * rotary)
    cos_sin = plain.positions_angles([max(n - 1, 0) for n in lengths], R).to(DEV) if R else None
    slots = [tables[t][(n - 1) // bs] * bs + (n - 1) % bs if n else -1 for t, n in enumerate(lengths)]
    slots[4] = -1
    positions, order, scale = i32([n - 1 for n in lengths]), i32([3, 1, 0, 2, 9, 8, 7, 6, 5, 4]), plain.default_scale(D)
    for store in (True, False):
        one, two = [x.clone() for x in cache], [x.clone() for x in cache]
        out = [torch.full((T, H, D), 7.0, dtype=BF16, device=DEV) for _ in range(2)]
        ops.attn_decode_fresh8(qkv, *gains, cos_sin, i32(slots), 1e-6, store, *one, positions, i32(tables), out[0], H, scale, window, 300, part_size=part,
                               order=order)  # fmt: skip
        q = torch.empty((T, H, D), dtype=BF16, device=DEV)
        kept = slots if store else [-1] * T
        ops.qk_norm_rope_store8(qkv, *gains, cos_sin, i32(kept), q, *two, H, KV, 1e-6, store_kv=store)
        ops.attn_single_query8(q, *two, order, positions, None, i32(tables), out[1], scale, window, 300, part_size=part)
        same = [t for t in range(T) if t != 4 or not store]  # token 4 attends itself, which two kernels cannot
        assert torch.equal(out[0][same], out[1][same]) and all(same_bytes(x, y) for x, y in zip(one, two))
        assert (out[0][9] == 0).all()
        if store:
            ops.qk_norm_rope_store8(qkv[4:5], *gains, None if cos_sin is None else cos_sin[4:5], i32([tables[4][32 // bs] * bs + 32 % bs]), q[4:5], *two,
                                    H, KV, 1e-6)  # fmt: skip
            ops.attn_single_query8(q, *two, order, positions, None, i32(tables), out[1], scale, window, 300, part_size=part)
            assert torch.equal(out[0][4], out[1][4])
