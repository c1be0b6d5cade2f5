"""The single-token operators on a B200 against plain implementations in 64 bits: block tables and slot maps, the
attention input side with several rotary axes, attention of one new token over the paged cache, and linear attention
with a decay for each head; then a run of them together, as a conversation makes it.

Tolerances: a rounding to bf16 is off by at most half a step, 2^-8 of the value; fp32 arithmetic adds 2^-24 per
operation of the sum of the terms' magnitudes, counted per test."""

from __future__ import annotations

import math

import pytest
import torch

from jeff_b200 import _lib, kernels
from jeff_b200 import constants as C
from jeff_b200.prefix_pool import FAST_PATH_SHAPES, PrefixPool

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8    # half a bf16 step, relative
ULP = 2.0 ** -24    # half an fp32 step, relative
FIXED = FAST_PATH_SHAPES.fixed_pages


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert _lib.device_status() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator("cuda").manual_seed(seed)


def normal(g: torch.Generator, *shape: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def close(got: torch.Tensor, want: torch.Tensor, tolerance: torch.Tensor) -> None:
    off = (got.double() - want).abs() - tolerance
    assert not torch.isnan(off).any()
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than it may be"


# ---------------------------------------------------------------- block tables and slot maps


def plain_tables(lengths, new, free, tables, kv_entry, tokens, page, fixed):
    """What block_tables does, one row after the other on the host."""
    tables = [list(r) for r in tables]
    width = len(tables[0])
    slots, rows, positions, starts, taken = [], [], [], [0], [0]
    at = 0
    for r, (have, add) in enumerate(zip(lengths, new)):
        have, add = max(have, 0), max(add, 0)

        def take():
            nonlocal at
            at += 1
            return free[at - 1] if at <= len(free) else 0

        if fixed and have == 0 and add > 0:
            for e in range(kv_entry):
                tables[r][e] = take()
        fresh = {}
        for j in range(min(-(-have // page), width - kv_entry), min(-(-(have + add) // page), width - kv_entry)):
            short = at >= len(free)
            tables[r][kv_entry + j] = take()
            if short:
                fresh[j] = True
        for pos in range(have, have + add):
            j = pos // page
            lost = j >= width - kv_entry or j in fresh
            slots.append(-1 if lost else tables[r][kv_entry + j] * page + pos % page)
            rows.append(r)
            positions.append(pos)
        starts.append(starts[-1] + add)
        taken.append(at)
    pad = max(0, tokens - len(slots))
    return (tables, (slots + [-1] * pad)[:tokens], (rows + [-1] * pad)[:tokens], (positions + [0] * pad)[:tokens],
            starts, taken)


@pytest.mark.parametrize(("lengths", "new", "spare", "entry", "width", "tokens", "page", "fixed"), [
    ([0], [1], 5, 0, 4, 1, 32, False),                                   # the smallest call
    ([31, 32, 33, 0, 64], [1, 1, 1, 1, 0], 10, 2, 9, 8, 32, False),      # before, at and past a page's end; a row idle
    ([0, 5, 0, 0], [40, 3, 0, 64], 30, 3, 8, 120, 32, True),             # fresh rows take their fixed pages too
    ([7, 0, 100], [70, 200, 1], 3, 1, 12, 300, 32, False),               # the free list runs out
    ([0, 60], [200, 100], 40, 2, 4, 300, 32, False),                     # rows past their tables
    ([-4, 3], [2, -7], 9, 1, 6, 5, 16, False),                           # negative counts are zero
    ([5, 6, 7], [30, 30, 30], 40, 1, 9, 50, 7, True),                    # fewer places than tokens; pages of 7
    ([3], [4], 0, 1, 5, 9, 4, False),                                    # an empty free list, one page needed
    ([i * 37 % 500 for i in range(1500)], [i % 4 for i in range(1500)], 900, 5, 30, 2500, 32, True),
    ([0] * 300, [i % 90 for i in range(300)], 40000, 50, 60, 16384, 32, True),
    ([2 ** 31 - 1, 0], [5, 2], 4, 1, 3, 9, 32, False),                   # a length at the type's end
])
def test_block_tables(lengths, new, spare, entry, width, tokens, page, fixed) -> None:
    b = len(lengths)
    filler = [[1000 + 70 * r + e for e in range(width)] for r in range(b)]
    free = [5 + 3 * i for i in range(spare)]
    if lengths[0] == 2 ** 31 - 1:
        new_plain = [0, 2]   # no position past the type's end exists
    else:
        new_plain = new
    want = plain_tables([min(x, 10 ** 6) for x in lengths], new_plain, free, filler, entry, tokens, page, fixed)
    wide = torch.full((b + 1, width + 3), -7, dtype=torch.int32, device="cuda")   # rows and entries behind: untouched
    wide[:b, :width] = i32(filler)
    tables = wide[:, :width]
    got = kernels.block_tables(i32(lengths), i32(new), i32(free), tables, entry, tokens, page_tokens=page, fixed=fixed)
    assert tables[:b].tolist() == want[0]
    assert bool((wide[b] == -7).all()) and bool((wide[:, width:] == -7).all())
    for name, x in zip(("slots", "rows", "positions", "starts", "taken"), want[1:]):
        assert getattr(got, name).tolist() == x, name


def test_block_tables_give_the_pools_own_order() -> None:
    """Fresh rows get the tables that PrefixPool.reserve gives them."""
    counts = [45, 1, 320, 64]
    pool = PrefixPool(400, "cuda", max_prefix_tokens=512)
    slots = [pool.reserve(0, f"p{i}", n) for i, n in enumerate(counts)]
    free = torch.arange(2, 400, dtype=torch.int32, device="cuda")
    tables = torch.zeros(4, pool.width, dtype=torch.int32, device="cuda")
    got = kernels.block_tables(i32([0] * 4), i32(counts), free, tables, FIXED, sum(counts), fixed=True)
    assert torch.equal(tables, pool.tables[torch.tensor(slots, device="cuda")])
    assert int(got.taken[-1]) == 400 - 2 - pool.free_page_count()


@pytest.mark.parametrize("giants", [1, 2])
def test_block_tables_counts_past_the_type(giants) -> None:
    """More rows than one round of the sums holds, and counts whose sum passes 31 and 32 bits in the first round: the
    tokens that fit are listed as ever, and nothing is written around them."""
    b, tokens, top = 1500, 2000, 2 ** 31 - 1
    new = [1] * b
    new[10:10 + giants] = [top] * giants
    wide = torch.full((5, tokens + 4096), -9, dtype=torch.int64, device="cuda")

    def inside(i: int, size: int, dtype: torch.dtype) -> torch.Tensor:
        return wide[i].view(dtype)[2048:2048 + size]

    out = kernels.SlotMap(inside(0, tokens, torch.int64), *(inside(1 + i, size, torch.int32) for i, size in
                                                            enumerate((tokens, tokens, b + 1, b + 1))))
    tables = torch.zeros(b, 4, dtype=torch.int32, device="cuda")
    guard = wide.clone()
    free = [3 + i for i in range(4 * b)]
    kernels.block_tables(i32([0] * b), i32(new), i32(free), tables, 0, tokens, out=out)
    assert sum(new[:1024]) in (2 ** 31 + 1022, 2 ** 32 + 1020)
    take = [min(-(-n // 32), 4) for n in new]
    want_tables, at = [], 0
    for n in take:
        want_tables.append(free[at:at + n] + [0] * (4 - n))
        at += n
    assert tables.tolist() == want_tables
    where = [(r, 0) for r in range(10)] + [(10, p) for p in range(tokens - 10)]
    assert out.rows.tolist() == [r for r, _ in where] and out.positions.tolist() == [p for _, p in where]
    assert out.slots.tolist() == [want_tables[r][p // 32] * 32 + p % 32 if p < 128 else -1 for r, p in where]
    sums = [0]
    for n in new:
        sums.append(sums[-1] + n)
    assert out.starts.tolist() == [min(s, top) for s in sums]
    assert out.taken.tolist() == [sum(take[:r]) for r in range(b + 1)]
    for i, (size, dtype) in enumerate(((tokens, torch.int64), (tokens, torch.int32), (tokens, torch.int32),
                                       (b + 1, torch.int32), (b + 1, torch.int32))):
        guard[i].view(dtype)[2048:2048 + size] = wide[i].view(dtype)[2048:2048 + size]
    assert torch.equal(wide, guard)


# ---------------------------------------------------------------- attention input side


def plain_prep(pr, q_w1, k_w1, inv_freq, positions, axis_of):
    t = pr.shape[0]
    x = pr[:, :C.ATTN_PROJ].double()
    q = x[:, :4096].view(t, 8, 512)[:, :, :256]
    k = x[:, 4096:4608].view(t, 2, 256)
    angle = positions[axis_of].T.double() * inv_freq.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]

    def head(y, w):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + C.EPS) * w.double()
        a, b = y[..., :32], y[..., 32:64]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., 64:]], -1)

    return head(q, q_w1), head(k, k_w1), pr[:, 4608:5120].view(t, 2, 256)


@pytest.mark.parametrize(("t", "sections", "interleaved", "reach"), [
    (1, (32,), False, 5), (3, (11, 11, 10), True, 100), (31, (8, 12, 12), False, 9000), (255, (11, 11, 10), True, 8192),
    (256, (32,), False, 8192), (257, (16, 8, 8), True, 8192),
    (64, (16, 16), False, 2 ** 31 - 1), (1000, (8, 8, 8, 8), True, 300000), (1217, (0, 32, 0), False, 60),
])
def test_attn_prep_axes(t, sections, interleaved, reach) -> None:
    g = gen(t)
    wide = normal(g, t, C.ATTN_PROJ + 24)
    pr = wide[:, :C.ATTN_PROJ + 8]   # a strided input
    if t > 2:
        pr[1] = 0                    # a token of zeros
        pr[2] *= 1e4
    q_w1, k_w1 = 1 + 0.2 * normal(g, 256, dtype=torch.float32), 1 + 0.2 * normal(g, 256, dtype=torch.float32)
    inv_freq = 1.0 / (C.ROPE_THETA ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    positions = torch.randint(-min(reach, 50), reach, (len(sections), t), generator=g, device="cuda").int()
    axes = kernels.rope_axes(sections, interleaved)
    of = torch.tensor([axes >> 2 * i & 3 for i in range(32)], device="cuda")
    q, k, v = plain_prep(pr, q_w1, k_w1, inv_freq, positions, of)
    pages = -(-t // 32) + 3
    kv = torch.full((pages, 3, 2, 32, 2, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    slots = torch.randperm(pages * 32, generator=g, device="cuda")[:t]
    slots[0] = -1                    # a token that is not kept
    if t > 4:
        slots[3], slots[4] = pages * 32, 2 ** 40   # slots past the pool are written nowhere
    kn, vn = (torch.empty(t, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    got = kernels.attn_prep_axes(pr, q_w1, k_w1, inv_freq, positions, axes, kn=kn, vn=vn, kv=kv, attn_layer=1,
                                 slots=slots)
    # the norm: 256 squares summed, a root and two products; the turn: two products and a sum; sine and cosine to 2^-21
    slack = 32 * ULP * 8
    for out, want in ((got, q), (kn, k)):
        top = want.abs().amax(-1, keepdim=True)
        close(out, want, HALF * want.abs() + slack * top)
    assert torch.equal(vn, v)
    want_kv = torch.full_like(kv, 7.0)
    for i, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * 32:
            want_kv[slot // 32, 1, 0, slot % 32] = kn[i]
            want_kv[slot // 32, 1, 1, slot % 32] = vn[i]
    assert torch.equal(kv, want_kv)
    only = torch.full_like(kv, 7.0)   # the pages alone, and kn and vn alone, give the same
    q2 = kernels.attn_prep_axes(pr, q_w1, k_w1, inv_freq, positions, axes, kv=only, attn_layer=1, slots=slots)
    assert torch.equal(only, kv) and torch.equal(q2, got)


def test_attn_prep_axes_shares_positions() -> None:
    """Text: one row of positions standing for all axes (expanded) is the same as its copies."""
    g = gen(3)
    pr, w = normal(g, 70, C.ATTN_PROJ), torch.ones(256, device="cuda")
    f = torch.rand(32, generator=g, device="cuda")
    one = torch.arange(70, dtype=torch.int32, device="cuda")
    axes = kernels.rope_axes([11, 11, 10], True)
    outs = []
    for positions in (one.expand(3, -1), one.repeat(3, 1)):
        kn, vn = (torch.empty(70, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        outs.append((kernels.attn_prep_axes(pr, w, w, f, positions, axes, kn=kn, vn=vn), kn, vn))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_attn_prep_axes_agrees_with_the_text_form() -> None:
    """With one axis it is attn_prep_rows up to that one's own rounding points: the norm's result, the sine and cosine,
    each product and the sum (half a step each, of values up to |a| + |b|)."""
    g = gen(5)
    t = 64
    pr = normal(g, t, C.ATTN_PROJ)
    w = 1 + 0.1 * normal(g, 256, dtype=torch.float32)
    inv_freq = 1.0 / (C.ROPE_THETA ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    kn, vn, kn2, vn2 = (torch.empty(t, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    rows = kernels.attn_prep_rows(pr, w, w, inv_freq, i32([40, 900]), kn, vn, 32)
    positions = torch.cat([torch.arange(40, 72), torch.arange(900, 932)]).int().cuda()[None]
    axes = kernels.attn_prep_axes(pr, w, w, inv_freq, positions, kernels.rope_axes((32,)), kn=kn2, vn=vn2)
    assert torch.equal(vn, vn2)
    for a, b in ((rows, axes), (kn, kn2)):
        x = torch.maximum(a[..., :32].float().abs(), a[..., 32:64].float().abs())
        size = torch.cat([2 * x, 2 * x, a[..., 64:].float().abs()], -1)
        close(a, b.double(), 5 * HALF * size + 900 * 2.0 ** -23)


def test_attn_prep_axes_refuses() -> None:
    w = torch.ones(256, device="cuda")
    f = torch.ones(32, device="cuda")
    pr = torch.zeros(3, C.ATTN_PROJ, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    kn = torch.empty(3, 2, 256, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(3, 6, 2, 32, 2, 256, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    call = lambda **kw: kernels.attn_prep_axes(**(dict(pr=pr, q_w1=w, k_w1=w, inv_freq=f, positions=pos,  # noqa: E731
                                                       axes=kernels.rope_axes((16, 16)), kn=kn, vn=kn.clone()) | kw))
    for over, says in (({"axes": kernels.rope_axes((11, 11, 10))}, "axis past"), ({"vn": None}, "keys and values"),
                       ({"kv": kv}, "keys and values"), ({"slots": slots}, "keys and values"),
                       ({"kv": kv[:, :, :, :16], "slots": slots}, "kv: expected"),
                       ({"kv": kv, "slots": slots, "attn_layer": 6}, "6 layers"),
                       ({"kv": kv[..., :128], "slots": slots}, "packed"),
                       ({"slots": slots.int(), "kv": kv}, "slots: expected"),
                       ({"positions": pos[:, :2]}, "positions: expected"), ({"q_w1": w[:255]}, "q_w1: expected"),
                       ({"pr": torch.cat([pr, pr[:, :1]], 1)}, "ldpr 5121")):
        with pytest.raises(ValueError, match=says):
            call(**over)


# ---------------------------------------------------------------- attention of one new token


def cache(g: torch.Generator, lengths: list[int], layers: int, layer: int, kv_heads: int, dim: int, entry: int,
          extra: int = 0, tail: float = math.nan):
    """A paged cache of these lengths, its pages in random order; what no token fills holds `tail`."""
    held = [-(-max(n, 0) // 32) for n in lengths]
    total = sum(held) + 3
    kv = torch.full((total, layers, 2, 32, kv_heads, dim), tail, dtype=torch.bfloat16, device="cuda")
    width = entry + max([*held, 1]) + extra
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    order = (torch.randperm(total - 3, generator=torch.Generator().manual_seed(len(lengths))) + 3).tolist()
    dense = []
    for r, n in enumerate(lengths):
        n = max(n, 0)
        mine = [order.pop() for _ in range(held[r])]
        tables[r, entry:entry + held[r]] = torch.tensor(mine, dtype=torch.int32)
        rows = normal(g, 2, n, kv_heads, dim)
        for j, page in enumerate(mine):
            part = rows[:, 32 * j:32 * j + 32]
            kv[page, layer, :, :part.shape[1]] = part
        dense.append(rows)
    return kv, tables.cuda(), dense


def plain_decode(q, dense, scale, pr=None):
    """(want, tolerance) in 64 bits. The scores' fp32 error is d + 2 operations on the magnitudes of their terms, and
    with the exponential's 2^-21 it moves a weight by that much relative to it, numerator and denominator alike; the
    weights may be held as two bf16 parts (2^-17), and the sums over the keys add an operation for each of 64 partial
    sums and one for each key that a warp adds."""
    b, heads, dim = q.shape
    want, tol = torch.zeros(b, heads, dim, dtype=torch.float64, device="cuda"), torch.zeros(
        b, heads, dim, dtype=torch.float64, device="cuda")
    for r, both in enumerate(dense):
        n = both.shape[1]
        if n == 0:
            continue
        group = heads // both.shape[2]
        k, v = (x.double().repeat_interleave(group, 1) for x in both)
        s = torch.einsum("hd,jhd->hj", q[r].double(), k) * scale
        size = torch.einsum("hd,jhd->hj", q[r].double().abs(), k.abs()) * abs(scale)
        p = torch.softmax(s, -1)
        want[r] = torch.einsum("hj,jhd->hd", p, v)
        moved = (dim + 2) * ULP * size.amax(-1, keepdim=True) + 2.0 ** -21 + 2.0 ** -17 + (64 + n / 4) * ULP
        tol[r] = 2 * moved * torch.einsum("hj,jhd->hd", p, v.abs())
    if pr is not None:
        gate = torch.sigmoid(pr[:, :2 * heads * dim].double().view(b, heads, 2, dim)[:, :, 1])
        want, tol = want * gate, (tol + 8 * ULP * want.abs()) * gate
    return want, HALF * want.abs() + tol + 1e-30


@pytest.mark.parametrize(("lengths", "heads", "kv_heads", "dim", "gated"), [
    ([1], 8, 2, 256, True),
    ([0, 1, 2, 31, 32, 33, 0, 63, 64, 65, 100], 8, 2, 256, True),
    ([1000], 8, 2, 256, False),
    ([8192, 5, 777, 0], 8, 2, 256, True),
    ([300, 17, 1025], 6, 2, 256, True),       # three query heads to a key/value head
    ([129, 16], 1, 1, 256, False),
    ([250, 47, 400, 3], 32, 8, 128, False),   # other head layouts
    ([500, 33], 16, 1, 128, True),            # sixteen query heads to one
    ([129, 700, 16], 9, 1, 256, True),
    ([64, 2000], 16, 1, 64, False),
    ([300, 5], 5, 1, 256, False),
    ([40, 41, 700], 5, 1, 64, False),
    ([99, 1500], 12, 12, 64, True),
    ([64] * 200, 8, 2, 256, False),           # more rows than SMs
    ([1] * 700, 14, 2, 64, True),
    ([20000], 2, 2, 128, False),
    ([77, 0, 3000, 16], 8, 8, 128, True),     # eight key/value heads side by side
    ([333, 48, 47], 40, 8, 64, False),
    ([15, 700, 130], 24, 6, 256, True),
    ([513, 90], 16, 16, 256, False),
    ([5, 40] * 600, 2, 1, 64, False),         # more rows than a CTA holds the lengths of
    ([5000, 7, 9000, 6000, 0, 12000, 6700], 8, 8, 64, True),   # many steps a share
    ([20000, 30000, 1, 27001], 8, 2, 256, True),
    ([3000, 2000] * 20, 32, 4, 128, False),
])
def test_decode_attention(lengths, heads, kv_heads, dim, gated) -> None:
    g = gen(sum(lengths) + heads)
    kv, tables, dense = cache(g, lengths, 3, 1, kv_heads, dim, entry=2)
    b = len(lengths)
    q = normal(g, b, heads + 1, dim)[:, :heads]   # rows apart
    pr = normal(g, b, 2 * heads * dim + 16) if gated else None
    got = kernels.decode_attention(q, kv, tables, 1, i32(lengths), 2, pr=pr)
    assert got.shape == ((b, heads * dim) if gated else (b, heads, dim))
    want, tol = plain_decode(q, dense, dim ** -0.5, pr)
    close(got.view(b, heads, dim), want, tol)
    again = kernels.decode_attention(q, kv, tables, 1, i32(lengths), 2, pr=pr)
    assert torch.equal(got, again)


def test_decode_attention_strided_pages_and_outputs() -> None:
    """A pool's own view (its pages far apart), an output inside a wider tensor, a scale of the caller's."""
    g = gen(9)
    lengths = [70, 45, 1, 0]
    pool = PrefixPool(300, "cuda")
    dense, slots = [], []
    for r, n in enumerate(lengths):
        slots.append(pool.reserve(0, str(r), n))
        rows = normal(g, 2, n, 2, 256)
        pages = pool.block_table(slots[-1])[FIXED:]
        for j, page in enumerate(pages):
            pool.kv[page, 4] = math.nan
            part = rows[:, 32 * j:32 * j + 32]
            pool.kv[page, 4, :, :part.shape[1]] = part
        dense.append(rows)
    tables = pool.tables[torch.tensor(slots, device="cuda")]
    q = normal(g, 4, 8, 256)
    wide = torch.full((4, 2048 + 32), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 16:2064].unflatten(1, (8, 256))
    kernels.decode_attention(q, pool.kv, tables, 4, i32(lengths), FIXED, scale=-0.11, out=out)
    want, tol = plain_decode(q, dense, -0.11)
    close(out, want, tol)
    assert bool((wide[:, :16] == 3).all()) and bool((wide[:, 2064:] == 3).all())


def test_decode_attention_large_scores() -> None:
    """Scores of both signs far beyond what an exponential holds, and a single key that takes all."""
    g = gen(10)
    lengths = [400, 129]
    kv, tables, dense = cache(g, lengths, 1, 0, 2, 256, entry=0)
    q = 64 * normal(g, 2, 8, 256)
    for x in dense:
        x[0, 100] = 30.0
    for r in range(2):
        kv[tables[r, 3], 0, 0, 4] = 30.0
    q[0] = q[0].abs()
    got = kernels.decode_attention(q, kv, tables, 0, i32(lengths), 0)
    want, tol = plain_decode(q, dense, 1 / 16)
    close(got, want, tol)


@pytest.mark.parametrize(("heads", "kv_heads", "dim"), [(8, 2, 256), (9, 3, 128), (16, 1, 64)])
def test_decode_attention_passes_nan_on(heads, kv_heads, dim) -> None:
    """A NaN in a query, a key or a value makes NaN of what the formula makes NaN of, in short rows as in cut ones, and
    of nothing else."""
    g = gen(12)
    lengths = [9000, 40, 9000, 40, 9000]
    kv, tables, dense = cache(g, lengths, 1, 0, kv_heads, dim, entry=0)
    q = normal(g, 5, heads, dim)
    q[0, 1, 3] = q[1, 0, 0] = math.nan
    for r, part, j in ((2, 0, 8000), (3, 0, 39), (4, 1, 17)):
        dense[r][part, j, kv_heads - 1, 5] = math.nan
        kv[tables[r, j // 32], 0, part, j % 32, kv_heads - 1, 5] = math.nan
    want, tol = plain_decode(q, dense, dim ** -0.5)
    got = kernels.decode_attention(q, kv, tables, 0, i32(lengths), 0)
    bad = want.isnan()
    assert bad.any(-1).sum() == 2 + 3 * (heads // kv_heads) and torch.equal(got.isnan(), bad)
    close(got[~bad], want[~bad], tol[~bad])


def test_decode_attention_bad_pages_and_lengths() -> None:
    """An entry outside the pool is no page: its tokens are left out. A length past the table's width is cut there,
    one below zero is none; a row whose pages are all bad is zeros."""
    g = gen(11)
    lengths = [200, 128, 96, 64]
    kv, tables, dense = cache(g, lengths, 2, 0, 2, 256, entry=1)
    tables[0, 1 + 2] = -3
    tables[0, 1 + 4] = kv.shape[0]
    tables[2, 1:] = 2 ** 31 - 1
    width = 1 + 4
    narrow = tables[:, :width]
    q = normal(g, 4, 8, 256)
    got = kernels.decode_attention(q, kv, narrow, 0, i32([200, 100000, 96, -5]), 1)
    keep = [j for j in range(128) if not 64 <= j < 96]
    seen = [dense[0][:, keep], dense[1][:, :128], dense[2][:, :0], dense[3][:, :0]]
    want, tol = plain_decode(q, seen, 1 / 16)
    close(got, want, tol)
    assert not got[2:].any()
    got = kernels.decode_attention(q, kv, tables, 0, i32(lengths), 1)
    keep = [j for j in range(200) if not (64 <= j < 96 or 128 <= j < 160)]
    want, tol = plain_decode(q, [dense[0][:, keep], dense[1], dense[2][:, :0], dense[3]], 1 / 16)
    close(got, want, tol)


def test_decode_attention_scratch_holds_anything() -> None:
    """The scratch needs no zeroing: NaN, ones in every bit, what other calls of the same and of other shapes left; a
    captured call replayed on it again and again gives the same bits."""
    g = gen(30)
    lengths = [1000, 3, 2500]
    kv, tables, dense = cache(g, lengths, 1, 0, 2, 256, entry=0)
    q, n = normal(g, 3, 8, 256), i32(lengths)
    scratch = torch.full((kernels._decode_scratch(16, 1, 256),), math.nan, device="cuda")
    want = kernels.decode_attention(q, kv, tables, 0, n, 0)
    close(want, *plain_decode(q, dense, 1 / 16))
    wide = normal(g, 3, 12, 256)
    for fill in (None, -1, 0, None, 2 ** 31 - 1):
        if fill is not None:
            scratch.view(torch.int32).fill_(fill)
        kernels.decode_attention(wide, kv, tables, 0, n, 0, scratch=scratch)
        assert torch.equal(kernels.decode_attention(q, kv, tables, 0, n, 0, scratch=scratch), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.decode_attention(q, kv, tables, 0, n, 0, scratch=scratch)
    for _ in range(5):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_decode_attention_far_pages() -> None:
    """A cache whose bytes pass 32 bits, its last page among those read."""
    g = gen(12)
    pages = (1 << 32) // (2 * 2 * 32 * 2 * 256) + 40   # 65,536 bytes a page of one layer: past 4 GB
    kv = torch.empty(pages, 1, 2, 32, 2, 256, dtype=torch.bfloat16, device="cuda")
    tables = i32([[pages - 1, 3, pages - 20]])
    rows = normal(g, 2, 90, 2, 256)
    for j, page in enumerate(tables[0].tolist()):
        kv[page, 0] = math.nan
        part = rows[:, 32 * j:32 * j + 32]
        kv[page, 0, :, :part.shape[1]] = part
    q = normal(g, 1, 8, 256)
    got = kernels.decode_attention(q, kv, tables, 0, i32([90]), 0)
    close(got, *plain_decode(q, [rows], 1 / 16))


def test_rows_left_short_of_pages_stay_without_them() -> None:
    """A row that found the free list empty holds the sink in its table: its later tokens on that page have no slot either,
    and its attention leaves the page out, whatever the sink holds."""
    g = gen(40)
    tables = torch.zeros(3, 6, dtype=torch.int32, device="cuda")
    tables[:, :3] = i32([[9, 9, 5], [9, 9, 6], [9, 9, 8]])
    lengths, new = i32([32, 32, 5]), i32([1, 1, 1])
    got = kernels.block_tables(lengths, new, i32([7]), tables, 2, 3)
    assert got.slots.tolist() == [7 * 32, -1, 8 * 32 + 5] and got.taken.tolist() == [0, 1, 2, 2]
    lengths += new
    got = kernels.block_tables(lengths, new, i32([]), tables, 2, 3)   # takes no page, so nothing else reports it
    assert got.slots.tolist() == [7 * 32 + 1, -1, 8 * 32 + 6] and got.taken.tolist() == [0, 0, 0, 0]
    assert got.positions.tolist() == [33, 33, 6] and tables[:, 2:].tolist() == [[5, 7, 0, 0], [6, 0, 0, 0], [8, 0, 0, 0]]
    kv = normal(g, 10, 2, 2, 32, 2, 256)
    q = normal(g, 3, 8, 256)
    y = kernels.decode_attention(q, kv, tables, 1, i32([34, 34, 7]), 2)
    dense = [torch.cat([kv[5, 1], kv[7, 1, :, :2]], 1), kv[6, 1], kv[8, 1, :, :7]]
    close(y, *plain_decode(q, dense, 1 / 16))


# ---------------------------------------------------------------- linear attention


def spots(tables: torch.Tensor, layer: int, heads: int, per: int):
    flat = layer * heads + torch.arange(heads, device="cuda")
    return tables[:, flat // per].long(), (flat % per).expand(tables.shape[0], -1)


def plain_linear(q, k, v, g, begin, real, beta=None):
    """(o, its terms' magnitudes, state, its terms' magnitudes) token by token in 64 bits."""
    b, n, heads, d = q.shape
    o, mag = (torch.zeros(b, n, heads, d, dtype=torch.float64, device="cuda") for _ in range(2))
    s, m = begin.double(), begin.double().abs()
    e = torch.exp(g.double()).expand(b, n, heads)
    for t in range(n):
        live = (t < real)[:, None, None, None]
        qt, kt, vt = (x[:, t].double() for x in (q, k, v))
        s1, m1 = e[:, t, :, None, None] * s, e[:, t, :, None, None] * m
        va = vt.abs()
        if beta is not None:
            bt = beta[:, t].double()[..., None]
            vt = bt * (vt - torch.einsum("bhij,bhi->bhj", s1, kt))
            va = bt * (va + torch.einsum("bhij,bhi->bhj", m1, kt.abs()))
        s = torch.where(live, s1 + kt[..., None] * vt[..., None, :], s)
        m = torch.where(live, m1 + kt.abs()[..., None] * va[..., None, :], m)
        o[:, t] = torch.where(live[..., 0], torch.einsum("bhij,bhi->bhj", s, qt) * d ** -0.5, 0.0)
        mag[:, t] = torch.where(live[..., 0], torch.einsum("bhij,bhi->bhj", m, qt.abs()) * d ** -0.5, 0.0)
    return o, mag, s, m


def linear_case(seed, b, n, heads, per, layer, kind):
    g = gen(seed)
    shape = (b, n, heads, 128)
    q, k = (torch.nn.functional.normalize(normal(g, *shape).float(), dim=-1).bfloat16() for _ in range(2))
    v = normal(g, *shape)
    if kind == "heads":
        decay = -0.5 * torch.rand(heads, generator=g, device="cuda")
    elif kind == "strong":
        decay = -30 * torch.rand(b, n, heads, generator=g, device="cuda")
    elif kind == "none":
        decay = torch.zeros(b, n, heads, device="cuda")
    else:
        decay = -torch.exp(2 * normal(g, b, n, heads, dtype=torch.float32) - 3)
        if kind == "resets":
            decay[torch.rand(b, n, heads, generator=g, device="cuda") < 0.05] = -math.inf
    width = (layer + 1) * heads // per + 3
    pages = 2 * b * width + 2
    state = torch.full((pages, per, 128, 128), 5.0, device="cuda")
    ids = (torch.randperm(pages - 2, generator=g, device="cuda") + 2).int().view(2, b, width)
    begin = 0.3 * normal(g, b, heads, 128, 128, dtype=torch.float32)
    page, slot = spots(ids[0], layer, heads, per)
    state[page, slot] = begin
    return q, k, v, decay, state, ids[0], ids[1], begin


SCANS = [
    (1, 1, 16, 6, 0, "mixed", None), (2, 2, 16, 6, 17, "mixed", None), (3, 63, 16, 6, 3, "mixed", (63, 1, 0)),
    (2, 64, 16, 6, 5, "resets", (64, 33)), (2, 65, 4, 4, 1, "heads", (65, 64)), (3, 127, 5, 2, 0, "strong", None),
    (2, 128, 16, 6, 2, "none", (128, 127)), (2, 129, 16, 6, 9, "resets", (129, 128)), (1, 300, 3, 1, 0, "mixed", None),
    (4, 257, 16, 6, 1, "mixed", (257, 0, 130, 256)), (1, 1000, 16, 6, 4, "heads", None), (20, 96, 16, 6, 0, "heads", None),
    (1, 1024, 2, 6, 0, "none", None), (2, 700, 1, 1, 3, "resets", (699, 700)),
]


@pytest.mark.parametrize(("b", "n", "heads", "per", "layer", "kind", "real"), SCANS)
def test_linear_scan(b, n, heads, per, layer, kind, real) -> None:
    q, k, v, g, state, tables, outs, begin = linear_case(b * 1000 + n, b, n, heads, per, layer, kind)
    lengths = i32(list(real) if real else [n] * b)
    before = state.clone()
    got = kernels.linear_scan(q, k, v, g, state, tables, layer, real=lengths if real else None, out_tables=outs)
    o, mag, s, m = plain_linear(q, k, v, g, begin, lengths)
    # a chunked form may round the probabilities and the state to bf16 ahead of their products (half a step of each
    # term) and the result once more; its sums add 128 terms a chunk and one a chunk
    close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)
    page, slot = spots(outs, layer, heads, per)
    ends = state[page, slot]
    # the state's terms: three bf16 parts of a decayed key (2^-24 of it), a decay factor to 2^-21, the sums
    close(ends, s, (2.0 ** -20 + (n / 4 + 64) * ULP) * m + 1e-30)
    assert float((ends.double() - s).norm()) <= 2.0 ** -19 * float(s.norm())
    before[page, slot] = ends
    assert torch.equal(state, before)   # nothing else is written
    for r, count in enumerate(lengths.tolist()):
        assert not got[r, count:].any()
    again = kernels.linear_scan(q, k, v, g, state, tables, layer, real=lengths if real else None)
    assert torch.equal(got, again) and torch.equal(state, before)


def test_linear_scan_strided_inputs_in_place() -> None:
    """q, k and v as parts of one projection, the decays as part of a wider tensor, the states updated in place."""
    b, n, heads = 2, 150, 16
    q, k, v, g, state, tables, _, begin = linear_case(7, b, n, heads, 6, 2, "mixed")
    wide = torch.cat([x.flatten(2) for x in (q, k, v)] + [q[..., 0, :24]], 2)
    parts = [wide[..., 2048 * i:2048 * i + 2048].unflatten(2, (16, 128)) for i in range(3)]
    gates = torch.cat([g, g + 1], 2)[..., :16]
    got = kernels.linear_scan(*parts, gates, state, tables, 2, out_tables=tables)
    o, mag, s, m = plain_linear(q, k, v, g, begin, i32([n] * b))
    close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)
    page, slot = spots(tables, 2, heads, 6)
    close(state[page, slot], s, (2.0 ** -20 + (n / 4 + 64) * ULP) * m + 1e-30)


def test_linear_scan_long_prompt_continues() -> None:
    """One long prompt at once gives what its two halves give one after the other (the tolerances of both)."""
    b, n, heads = 1, 4099, 16
    q, k, v, g, state, tables, outs, begin = linear_case(8, b, n, heads, 6, 1, "mixed")
    whole = kernels.linear_scan(q, k, v, g, state, tables, 1, out_tables=outs)
    page, slot = spots(outs, 1, heads, 6)
    end = state[page, slot].clone()
    cut = 2050
    one = kernels.linear_scan(q[:, :cut], k[:, :cut], v[:, :cut], g[:, :cut], state, tables, 1, out_tables=outs)
    two = kernels.linear_scan(q[:, cut:], k[:, cut:], v[:, cut:], g[:, cut:], state, outs, 1, out_tables=outs)
    o, mag, s, m = plain_linear(q, k, v, g, begin, i32([n]))
    both = torch.cat([one, two], 1)
    for got in (whole, both):
        close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)
    for got in (end, state[page, slot]):
        close(got, s, (2.0 ** -20 + (n / 4 + 64) * ULP) * m + 1e-30)


def test_linear_scan_broadcast_inputs() -> None:
    """One key and value row for all rows, one token for all tokens, decays of one row for all (strides of zero)."""
    q, k, v, g, state, tables, _, begin = linear_case(13, 3, 70, 2, 2, 0, "mixed")
    for kk, vv, gg in ((k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), g[:1].expand(3, -1, -1)),
                       (k[:, :1].expand(-1, 70, -1, -1), v, g[:, :1].expand(-1, 70, -1))):
        got = kernels.linear_scan(q, kk, vv, gg, state, tables, 0)
        o, mag, _, _ = plain_linear(q, kk, vv, gg, begin, i32([70] * 3))
        close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)


@pytest.mark.parametrize(("b", "n", "heads"), [(1, 700, 16), (5, 130, 16)])
def test_linear_scan_padding_holds_anything(b, n, heads) -> None:
    """What stands past a row's end, NaN in q, k, v and g, changes nothing."""
    q, k, v, g, state, tables, outs, _ = linear_case(14, b, n, heads, 6, 1, "mixed")
    real = [n - 1 - 37 * r for r in range(b)]
    want = kernels.linear_scan(q, k, v, g, state, tables, 1, real=i32(real), out_tables=outs)
    page, slot = spots(outs, 1, heads, 6)
    ends = state[page, slot].clone()
    for r, count in enumerate(real):
        for x in (q, k, v, g):
            x[r, count:] = math.nan
    got = kernels.linear_scan(q, k, v, g, state, tables, 1, real=i32(real), out_tables=outs)
    assert torch.equal(got, want) and torch.equal(state[page, slot], ends)


def test_linear_scan_captured() -> None:
    """A captured scan of a long prompt, replayed on other inputs, gives the eager bits."""
    q, k, v, g, state, tables, outs, _ = linear_case(15, 2, 600, 16, 6, 0, "mixed")
    page, slot = spots(outs, 0, 16, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = kernels.linear_scan(q, k, v, g, state, tables, 0, out_tables=outs)
    for scale in (0.5, -2.0):
        v *= scale
        want = kernels.linear_scan(q, k, v, g, state, tables, 0, out_tables=outs).clone()
        ends = state[page, slot].clone()
        state[page, slot] = 0
        graph.replay()
        assert torch.equal(o, want) and torch.equal(state[page, slot], ends)


def test_linear_bad_pages() -> None:
    """An entry outside the pool reads as zeros and is not written; the reserved pages are never written."""
    q, k, v, g, state, tables, outs, begin = linear_case(9, 3, 40, 6, 6, 0, "mixed")
    tables[0, 0] = -1
    tables[1, 0] = state.shape[0]
    outs[0, 0], outs[1, 0], outs[2, 0] = 1, 2 ** 31 - 1, 0
    before = state.clone()
    begin[:2] = 0
    got = kernels.linear_scan(q, k, v, g, state, tables, 0, out_tables=outs)
    o, mag, _, _ = plain_linear(q, k, v, g, begin, i32([40] * 3))
    close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)
    assert torch.equal(state, before)
    first = kernels.linear_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, tables, 0, out_tables=outs)
    close(first, o[:, 0], HALF * o[:, 0].abs() + (HALF + 2.0 ** -13) * mag[:, 0])
    assert torch.equal(state, before)


@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize(("b", "heads", "per", "layer", "kind"), [
    (1, 16, 6, 0, "mixed"), (5, 16, 6, 17, "mixed"), (3, 5, 2, 1, "resets"), (64, 16, 6, 3, "heads"),
    (2, 1, 1, 4, "strong"), (40, 3, 4, 2, "none"),
])
def test_linear_step(b, heads, per, layer, kind, delta) -> None:
    q, k, v, g, state, tables, outs, begin = linear_case(b + 50, b, 1, heads, per, layer, kind)
    beta = torch.sigmoid(normal(gen(b), b, 1, heads, dtype=torch.float32)).bfloat16() if delta else None
    o, mag, s, m = plain_linear(q, k, v, g, begin, i32([1] * b), beta)
    page, slot = spots(tables, layer, heads, per)
    opage, oslot = spots(outs, layer, heads, per)
    one = g if g.dim() == 1 else g[:, 0]
    for target in (outs, None):
        before = state.clone()
        got = kernels.linear_step(q[:, 0], k[:, 0], v[:, 0], one, state, tables, layer,
                                  beta=None if beta is None else beta[:, 0], out_tables=target)
        # two sums of 128 terms (three with beta), a decay factor to 2^-22
        close(got, o[:, 0], HALF * o[:, 0].abs() + (300 * ULP + 2.0 ** -21) * mag[:, 0])
        at = (opage, oslot) if target is not None else (page, slot)
        close(state[at], s, (140 * ULP + 2.0 ** -21) * m + 1e-30)
        before[at] = state[at]
        assert torch.equal(state, before)


def test_linear_refusals() -> None:
    q, k, v, g, state, tables, outs, _ = linear_case(3, 2, 8, 16, 6, 0, "mixed")
    for over, says in (({"k": k[:, :7]}, "k: expected"), ({"v": v.float()}, "v: expected"),
                       ({"g": g[..., :15]}, "g: expected"), ({"g": g.bfloat16()}, "g: expected"),
                       ({"state": state[..., :64]}, "state: expected"), ({"layer": -1}, "layer -1"),
                       ({"layer": 1}, "tables: expected"), ({"tables": tables[:1]}, "tables: expected"),
                       ({"out_tables": outs.long()}, "out_tables: expected"),
                       ({"real": i32([1, 2, 3])}, "real: expected"),
                       ({"out": torch.empty(2, 8, 2048, device="cuda")}, "out: expected"),
                       ({"q": q.transpose(2, 3).contiguous().transpose(2, 3)}, "packed")):
        with pytest.raises(ValueError, match=says):
            kernels.linear_scan(**(dict(q=q, k=k, v=v, g=g, state=state, tables=tables[:, :4], layer=0) | over))
    with pytest.raises(ValueError, match="beta: expected"):
        kernels.linear_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, tables, 0, beta=g[:, 0])


def test_linear_scan_padding_past_32_bits() -> None:
    """A row so long that its padding's 16-byte pieces pass 31 bits: zeros out past its end, and nothing around them."""
    n, real = 2 ** 27 + 4096, 2 ** 27 + 1000
    x = torch.zeros(1, n, 1, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.ones(n + 128, 1, 128, dtype=torch.bfloat16, device="cuda")
    state = torch.full((4, 1, 128, 128), 2.0, device="cuda")
    kernels.linear_scan(x, x, x, torch.zeros(1, device="cuda"), state, i32([[2]]), 0, real=i32([real]),
                        out_tables=i32([[3]]), out=out[64:64 + n][None])
    assert bool((out[:64] == 1).all()) and bool((out[64 + n:] == 1).all())
    assert not out[64 + real - 3000:64 + n].any() and not out[64:10064].any()
    assert torch.equal(state[3], state[2])
    del x, out
    torch.cuda.empty_cache()   # 69 GB


@pytest.mark.parametrize("n", [1, 5, 40, 700])
def test_linear_states_in_the_sink_read_as_zeros(n) -> None:
    """A fresh row that found no page for its state starts from zeros, whatever the sink holds; other rows are as ever."""
    q, k, v, g, state, tables, outs, begin = linear_case(16, 2, n, 6, 6, 0, "mixed")
    tables[0, 0] = 0
    state[0] = math.nan
    begin[0] = 0
    o, mag, s, m = plain_linear(q, k, v, g, begin, i32([n] * 2))
    got = kernels.linear_scan(q, k, v, g, state, tables, 0, out_tables=outs)
    close(got, o, HALF * o.abs() + (HALF + 2.0 ** -13) * mag)
    page, slot = spots(outs, 0, 6, 6)
    close(state[page, slot], s, (2.0 ** -20 + (n / 4 + 64) * ULP) * m + 1e-30)
    if n == 1:
        got = kernels.linear_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, tables, 0, out_tables=outs)
        close(got, o[:, 0], HALF * o[:, 0].abs() + (300 * ULP + 2.0 ** -21) * mag[:, 0])


@pytest.mark.parametrize("real", [False, True])
@pytest.mark.parametrize(("b", "n", "heads"), [(2, 5, 16), (2, 100, 3), (20, 130, 16), (1, 700, 16), (2, 1001, 2)])
def test_linear_scan_passes_what_is_not_finite_on(b, n, heads, real) -> None:
    """A value, key, query or decay that is not finite spoils what the recurrence spoils, the outputs from its token on
    and its entries of the state, and no earlier token's output, other column or head."""
    q, k, v, g, state, tables, outs, begin = linear_case(17, b, n, heads, 6, 0, "mixed")
    last = n - 2 if real else n
    at = n // 2 + 1   # the middle of a chunk
    h = heads - 1
    v[0, at, 0, 7] = math.nan
    v[b - 1, at + 1, 1, 100] = math.inf
    v[0, last - 1, 1, 127] = -math.inf
    q[0, at - 1, 0, 3] = math.nan
    if heads > 2:
        k[0, at, 2, 9] = math.nan
        k[b - 1, last - 1, 2, 60] = math.inf
    if heads > 5:
        g[0, at, h] = math.nan
        k[0, 3, h - 1, 100] = -math.inf
        v[b - 1, n // 3:n // 3 + 2, h - 2, :64] = -math.inf
    lengths = i32([last] * b)
    o, _, s, _ = plain_linear(q, k, v, g, begin, lengths)
    clean = [torch.where(x.isfinite(), x, 1) for x in (q, k, v, g)]
    _, mag, _, m = plain_linear(*clean, begin, lengths)
    got = kernels.linear_scan(q, k, v, g, state, tables, 0, real=lengths if real else None, out_tables=outs)
    page, slot = spots(outs, 0, heads, 6)
    ends = state[page, slot]
    assert not o.isfinite().all() and not s.isfinite().all()
    assert torch.equal(got.isfinite(), o.isfinite()) and torch.equal(ends.isfinite(), s.isfinite())
    fine = o.isfinite()
    close(got[fine], o[fine], (HALF * o.abs() + (HALF + 2.0 ** -13) * mag)[fine])
    fine = s.isfinite()
    close(ends[fine], s[fine], ((2.0 ** -20 + (n / 4 + 64) * ULP) * m + 1e-30)[fine])


def one_row(t: torch.Tensor, stride: int) -> torch.Tensor:
    """`t`, one row long, with `stride` between its rows: what a transposed or narrowed tensor may bring."""
    return torch.as_strided(t, t.shape, (stride, *t.stride()[1:]), t.storage_offset())


def test_one_row_with_any_stride() -> None:
    """The stride of a dimension of one says nothing: a single row, page, token or table is taken as it stands."""
    g = gen(41)
    kv, tables, dense = cache(g, [70], 2, 1, 2, 256, entry=1)
    q, pr, n = normal(g, 8, 1, 256).transpose(0, 1), normal(g, 1, 4096 + 8), i32([70])
    assert q.is_contiguous() and q.stride(0) == 256
    want, tol = plain_decode(q, dense, 1 / 16, pr)
    for stride in (0, 1, 5):
        out = one_row(torch.empty(1, 2048, dtype=torch.bfloat16, device="cuda"), stride)
        kernels.decode_attention(q, kv, one_row(tables, stride), 1, n, 1, pr=one_row(pr, stride), out=out)
        close(out.view(1, 8, 256), want, tol)
        close(kernels.decode_attention(one_row(q, stride), one_row(kv[2:3], stride), tables * 0 + 5, 1, n, 1), want * 0,
              tol * 0)   # a pool of one page, which the table does not name

        w, f = torch.ones(256, device="cuda"), torch.ones(32, device="cuda")
        x = normal(g, 1, C.ATTN_PROJ)
        pages = [torch.zeros(1, 2, 2, 32, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        slot, axes = torch.tensor([3], device="cuda"), kernels.rope_axes((32,))
        a = kernels.attn_prep_axes(x, w, w, f, i32([[9]]), axes, kv=pages[0], slots=slot)
        b = kernels.attn_prep_axes(one_row(x, stride), w, w, f, one_row(i32([[9]]), stride), axes,
                                   kv=one_row(pages[1], stride), slots=slot)
        assert torch.equal(a, b) and torch.equal(*pages)

        table = i32([[1, 2, 3, 0]])
        made = kernels.block_tables(i32([33]), i32([40]), i32([8]), one_row(table, stride), 1, 40)
        assert table.tolist() == [[1, 2, 3, 8]] and made.slots.tolist() == [3 * 32 + i for i in range(1, 32)] + [
            8 * 32 + i for i in range(9)]

        for tokens in (1, 4, 70, 1001):
            lq, lk, lv, decay, state, ids, outs, _ = linear_case(18, 1, tokens, 6, 6, 0, "mixed")
            page = int(outs[0, 0])
            o = kernels.linear_scan(lq, lk, lv, decay, state, ids, 0, out_tables=outs)
            end = state[page].clone()
            o2 = kernels.linear_scan(*(one_row(y, stride) for y in (lq, lk, lv, decay)), state, one_row(ids, stride), 0,
                                     out_tables=one_row(outs, stride))
            assert torch.equal(o, o2) and torch.equal(state[page], end)
        token = [y[:, 0] for y in (lq, lk, lv, decay)]
        o = kernels.linear_step(*token, state, ids, 0, out_tables=outs)
        o2 = kernels.linear_step(*(one_row(y, stride) for y in token), state, one_row(ids, stride), 0,
                                 out_tables=one_row(outs, stride))
        assert torch.equal(o, o2)
        one = [y.unsqueeze(1) for y in token]   # one token of one row, both strides free
        o3 = kernels.linear_scan(*(torch.as_strided(y, y.shape, (stride, 3, *y.stride()[2:]), y.storage_offset())
                                   for y in one), state, ids, 0)
        close(o3[:, 0], o.double(), 2 * HALF * o.double().abs() + 1e-5)


def test_linear_scan_counts_its_launches() -> None:
    """Rows in segments are three launches and need a scratch; inputs that go token by token, one key, value or query
    standing for all, are one and need none."""
    q, k, v, g, state, tables, _, _ = linear_case(19, 1, 700, 4, 4, 0, "mixed")
    two = linear_case(20, 2, 700, 4, 4, 0, "mixed")

    def made(*args, **kw) -> int:
        before = _lib.launches
        kernels.linear_scan(*args, 0, **kw)
        return _lib.launches - before

    none = torch.empty(0, device="cuda")
    assert made(q, k, v, g, state, tables) == 3
    assert made(q, k[:, :1].expand(-1, 700, -1, -1), v, g, state, tables, scratch=none) == 1
    assert made(two[0], two[1], two[2][:1].expand(2, -1, -1, -1), *two[3:6], scratch=none) == 1
    assert made(q[:, :7], k[:, :7], v[:, :7], g[:, :7], state, tables, scratch=none) == 1
    assert made(q.expand(1, -1, -1, -1), k, v, g, state, tables) == 3
    with pytest.raises(ValueError, match="a scratch of 0 floats"):
        made(q, k, v, g, state, tables, scratch=none)


@pytest.mark.parametrize(("b", "n", "heads", "kind"), [(30, 192, 16, "heads"), (2, 2000, 16, "mixed")])
def test_linear_scan_errors_do_not_lean(b, n, heads, kind) -> None:
    """The outputs' errors are roundings, which lean to neither side, while a factor that is off by 2^-9 throughout leans.
    With no negative number anywhere nothing cancels: along a chunk's outputs, the errors' projection has a variance of at
    most (2^-8)^2 / 3 for each rounding of its terms, of the scores and of the state's copy, at the worst one rounding of
    each shared by all. The mean over all rows' heads' chunks stays within six deviations, and 2^-13 for sums that cut off."""
    q, k, v, g, state, tables, _, _ = linear_case(23, b, n, heads, 6, 0, kind)
    q, k, v = q.abs(), k.abs(), v.abs()
    state.abs_()
    page, slot = spots(tables, 0, heads, 6)
    got = kernels.linear_scan(q, k, v, g, state, tables, 0)
    o, _, _, _ = plain_linear(q, k, v, g, state[page, slot], i32([n] * b))
    lean = torch.stack([(x * y).sum((1, 3)) / (y * y).sum((1, 3)) for x, y in zip((got.double() - o).split(64, 1),
                                                                                  o.split(64, 1))])
    bound = 6 * HALF * (2 / 3 / lean.numel()) ** 0.5 + 2.0 ** -13
    assert bound < 2.0 ** -10
    assert abs(float(lean.mean())) <= bound


# ---------------------------------------------------------------- together


def test_a_conversation() -> None:
    """Three requests of mixed lengths: block tables for their prompts, the prompts' keys and values into the pages and
    their recurrent states, then tokens one by one: new slots, the token's keys and values, its attention over the whole
    cache and its step of the recurrent state. The steps run once eagerly and once as one captured graph replayed, with
    the same bits, each step's outputs against 64 bits. A fourth row is idle throughout."""
    g = gen(77)
    pool = PrefixPool(500, "cuda", max_prefix_tokens=256)
    b, prompts, steps, attn, lin = 4, [45, 31, 96, 0], 4, 2, 7
    free = torch.arange(2, 500, dtype=torch.int32, device="cuda")
    tables = torch.zeros(b, pool.width, dtype=torch.int32, device="cuda")
    fill = sum(prompts) + 5
    m = kernels.block_tables(i32([0] * b), i32(prompts), free, tables, FIXED, fill, fixed=True)
    left = free[int(m.taken[-1]):]
    w = torch.ones(256, device="cuda")
    inv_freq = 1.0 / (C.ROPE_THETA ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    axes = kernels.rope_axes((11, 11, 10), True)
    pool.kv[2:] = math.nan   # what nothing has written; the reserved page of zeros stays

    pr = normal(g, fill, C.ATTN_PROJ)
    kn, vn = (torch.empty(fill, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kernels.attn_prep_axes(pr, w, w, inv_freq, m.positions.expand(3, -1).contiguous(), axes, kn=kn, vn=vn, kv=pool.kv,
                           attn_layer=attn, slots=m.slots)
    bounds = m.starts.tolist()
    dense = [torch.stack([kn[bounds[r]:bounds[r + 1]], vn[bounds[r]:bounds[r + 1]]]) for r in range(b)]

    n = max(prompts) + steps
    q, k = (torch.nn.functional.normalize(normal(g, b, n, 16, 128).float(), dim=-1).bfloat16() for _ in range(2))
    v, decay = normal(g, b, n, 16, 128), -0.2 * torch.rand(b, n, 16, generator=g, device="cuda")
    zeros = torch.ones(b, pool.width, dtype=torch.int32, device="cuda")   # the empty prefix: the page of zeros
    real = i32(prompts)
    page, slot = spots(tables, lin, 16, 6)
    kernels.linear_scan(q[:, :96], k[:, :96], v[:, :96], decay[:, :96], pool.state, zeros, lin, real=real,
                        out_tables=tables)
    o, mag, _, _ = plain_linear(*(torch.stack([torch.cat([x[r, :prompts[r]], x[r, 96:], x[r, prompts[r]:96]])
                                               for r in range(b)]) for x in (q, k, v, decay)),
                                torch.zeros(b, 16, 128, 128, device="cuda"), i32([p + steps if p else 0 for p in prompts]))

    new = i32([1, 1, 1, 0])
    lengths, held = i32(prompts), left.clone()
    step_pr = normal(g, steps, b, C.ATTN_PROJ)
    x = {"pr": step_pr[0].clone(), "q": q[:, 96].clone(), "k": k[:, 96].clone(), "v": v[:, 96].clone(),
         "g": decay[:, 96].clone()}
    start = (lengths.clone(), tables.clone(), pool.data.clone(), held.clone())

    def step():
        mm = kernels.block_tables(lengths, new, held, tables, FIXED, b)
        # the rows' tokens are packed in row order and the idle row is the last: token i is row i's
        aq = kernels.attn_prep_axes(x["pr"], w, w, inv_freq, mm.positions.expand(3, -1).contiguous(), axes,
                                    kv=pool.kv, attn_layer=attn, slots=mm.slots)
        lengths.add_(new)
        y = kernels.decode_attention(aq, pool.kv, tables, attn, lengths, FIXED, pr=x["pr"])
        lo = kernels.linear_step(x["q"], x["k"], x["v"], x["g"], pool.state, tables, lin)
        # the pages taken leave the front of the free list
        held.copy_(held[(torch.arange(len(held), device="cuda") + mm.taken[-1]) % len(held)])
        return aq, y, lo

    def reset():
        for target, source in zip((lengths, tables, pool.data, held), start):
            target.copy_(source)

    eager = []
    for t in range(steps):
        for name, source in (("pr", step_pr[t]), ("q", q[:, 96 + t]), ("k", k[:, 96 + t]), ("v", v[:, 96 + t]),
                             ("g", decay[:, 96 + t])):
            x[name].copy_(source)
        aq, y, lo = step()
        eager.append((aq, y, lo))
        for r in range(3):
            assert int(lengths[r]) == prompts[r] + t + 1
            last = int(lengths[r]) - 1
            mine = pool.kv[int(tables[r, FIXED + last // 32]), attn, :, last % 32]
            dense[r] = torch.cat([dense[r], mine[:, None]], 1)
        want, tol = plain_decode(aq, dense, 1 / 16, x["pr"])
        close(y.view(b, 8, 256), want, tol)
        for r in range(3):
            i = prompts[r] + t
            close(lo[r], o[r, i], HALF * o[r, i].abs() + 2.0 ** -13 * mag[r, i])
    reset()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    reset()
    for t in range(steps):
        for name, source in (("pr", step_pr[t]), ("q", q[:, 96 + t]), ("k", k[:, 96 + t]), ("v", v[:, 96 + t]),
                             ("g", decay[:, 96 + t])):
            x[name].copy_(source)
        graph.replay()
        for a, e in zip(outs, eager[t]):
            assert torch.equal(a[:3], e[:3])


def test_on_a_stream_of_its_own() -> None:
    """Work on two streams at once, each with its own inputs, gives what one stream gives."""
    g = gen(21)
    lengths = [900, 64, 300]
    kv, tables, _ = cache(g, lengths, 1, 0, 2, 256, entry=0)
    cases = [normal(g, 3, 8, 256) for _ in range(8)]
    want = [kernels.decode_attention(q, kv, tables, 0, i32(lengths), 0) for q in cases]
    n = i32(lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(cases):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kernels.decode_attention(q, kv, tables, 0, n, 0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_at_once_on_three_streams() -> None:
    """Scans in segments and whole, steps and decode attention at once give what each gives alone."""
    g = gen(22)
    long, short = linear_case(1, 1, 1001, 16, 6, 0, "tokens"), linear_case(2, 40, 128, 16, 6, 0, "tokens")
    lengths = [5000, 1, 3000, 64]
    kv, tables, _ = cache(g, lengths, 2, 1, 2, 256, entry=0)
    q, n = normal(g, 4, 8, 256), i32(lengths)

    def scan(case):
        q, k, v, decay, state, ids, out_ids, _ = case
        return kernels.linear_scan(q, k, v, decay, state, ids, 0, out_tables=out_ids)

    work = [lambda: scan(long), lambda: scan(short), lambda: kernels.decode_attention(q, kv, tables, 1, n, 0)]
    want = [f() for f in work]
    torch.cuda.synchronize()
    finals = [case[4].clone() for case in (long, short)]
    streams = [torch.cuda.Stream() for _ in work]
    got = []
    for _ in range(10):
        for f, stream in zip(work, streams):
            with torch.cuda.stream(stream):
                got.append(f())
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 3])
    assert all(torch.equal(a, b[4]) for a, b in zip(finals, (long, short)))


def test_scans_in_a_row_in_place() -> None:
    """Scans that each go on from the state that the one before left in the same pages, launched without a wait in
    between and replayed as a graph, give what they give one at a time."""
    q, k, v, decay, state, ids, _, _ = linear_case(3, 1, 1001, 16, 6, 1, "tokens")
    start = state.clone()
    cut = [300, 1001, 700]

    def run(wait: bool) -> list[torch.Tensor]:
        state.copy_(start)
        outs = []
        for n in cut:
            outs.append(kernels.linear_scan(q[:, :n], k[:, :n], v[:, :n], decay[:, :n], state, ids, 1, out_tables=ids))
            outs.append(kernels.linear_step(q[:, n - 1], k[:, n - 1], v[:, n - 1], decay[:, n - 1], state, ids, 1))
            if wait:
                torch.cuda.synchronize()
        return outs + [state.clone()]

    want = run(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(False)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
