"""GPU: paged append, paged attention with a shared prefix and token log
probabilities through the Python mirror of the C-ABI, against plain 64-bit
forms (serving_ref.py, which derives the bounds)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import serving_ref as ref
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def within(got, want, bound, what):
    got, want = got.double().cpu(), want.cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= bound.cpu() + 1e-30)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[bad][0]} for {want[bad][0]}, bound {bound.cpu().expand_as(got)[bad][0]}"


# ---------------------------------------------------------------- append ---

SHAPES = [(9, 3, 64), (32, 8, 128), (8, 1, 128), (4, 4, 64), (16, 1, 64)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_append(yl, torch_cuda, dtype, half, shape):
    """New rows of sequences of uneven lengths (an idle slot, a first token, a chunk that crosses pages), behind them
    padding rows that are left alone, like every other slot of the pool."""
    t = DTYPES[dtype]
    g = ref.Geometry(1, *shape, page=16, lens=[1, 40, 7, 33, 16], rows=[1, 19, 0, 1, 16], pad_rows=3)
    k, v = g.pool(t)
    qkv = torch.from_numpy(g.rng.standard_normal((g.n_rows, (g.heads + 2 * g.kv) * g.hd))).float()
    cs = ref.rope_cs(64, g.hd)
    want = ref.append(g, qkv, k, v, cs, half)
    kd, vd = k.cuda(), v.cuda()
    q = torch.full((g.n_rows, g.heads, g.hd), 7.0, dtype=t, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    yl.paged_append(qkv.cuda(), yl.KvPages.of(kd, vd), g.device(yl, status), g.heads, rope_cs=cs.cuda(),
                    rope_mode=yl.ROPE_LLAMA3 if half else yl.ROPE_GGUF, q_out=q)
    assert status.item() == 0
    new = int(g.row_start[-1])
    assert (q[new:] == 7.0).all()
    for got, w, b, what in ((q[:new], want[0][:new], want[3][:new], "q"), (kd, want[1], want[4], "k"),
                            (vd, want[2], want[5], "v")):
        within(got, w, b + (w.abs() + b) * ref.half_step(t) + 2.0**-25 * (t == torch.float16), what)
    for pool, before in ((kd, k), (vd, v)):  # untouched slots keep their bits
        untouched = torch.ones(g.n_pages, g.page, dtype=torch.bool)
        for i in range(len(g.lens)):
            for p in g.positions(i):
                untouched[int(g.table[i, p // g.page]), int(p % g.page)] = False
        assert torch.equal(pool.cpu()[untouched], before[untouched])


def test_append_without_rotation_or_queries(yl, torch_cuda):
    """rope_cs None copies; q_out None leaves the query heads of the rows alone; qkv rows further apart than a row."""
    g = ref.Geometry(2, 8, 2, 64, page=8, lens=[20, 3], rows=[9, 3])
    wide = torch.from_numpy(g.rng.standard_normal((g.n_rows, 12 * 64 + 32))).float()
    qkv = wide[:, : 12 * 64]
    for t in DTYPES.values():
        k, v = g.pool(t)
        want = ref.append(g, qkv.contiguous(), k, v, None, False)
        kd, vd = k.cuda(), v.cuda()
        yl.paged_append(wide.cuda()[:, : 12 * 64], yl.KvPages.of(kd, vd), g.device(yl), 8)
        assert torch.equal(kd.cpu().double(), want[1].to(t).double())
        assert torch.equal(vd.cpu().double(), want[2].to(t).double())


def test_append_reports_bad_positions(yl, torch_cuda):
    """A page id that is no page, a position without a table slot, one beyond the rotation table and a row before
    position 0: the others are written, these are not, and the status word says so."""
    hd = 64
    for kind in ("page", "slot", "rope", "before"):
        g = ref.Geometry(3, 4, 2, hd, page=8, lens=[12, 24], rows=[3, 2], spare_slots=0)
        k, v = g.pool(torch.float32)
        qkv = torch.from_numpy(g.rng.standard_normal((5, 8 * hd))).float()
        n_cs = 32
        bad = [3, 4]
        if kind == "page":
            g.table[1, 2] = g.n_pages
        elif kind == "slot":
            g.table = g.table[:, :2].copy()
        elif kind == "rope":
            n_cs = 22
        else:
            g.lens[1], bad = 1, [3]
        kd, vd = k.cuda(), v.cuda()
        q = torch.full((5, 4, hd), 7.0, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        yl.paged_append(qkv.cuda(), yl.KvPages.of(kd, vd), g.device(yl, status), 4, rope_cs=ref.rope_cs(n_cs, hd).cuda(),
                        q_out=q)
        assert status.item() == -6, kind
        changed = (kd.cpu() != k).any(-1).any(-1)
        assert int(changed.sum()) == 5 - len(bad), kind
        if kind in ("rope", "before"):  # no position, no rotation
            assert (q[bad] == 7.0).all() and not (q[:3] == 7.0).any(), kind
        else:  # the row has a position: its query is rotated
            assert not (q == 7.0).any(), kind


# ------------------------------------------------------------- attention ---

@pytest.fixture
def own_pass(yl):
    """A shared prefix gets a pass of its own however short it is."""
    yl.config_set("paged_share", 1)
    yield
    yl.config_set("paged_share", -1)

def attend(yl, g, q, k, v, scale, out_dtype=None, shared=None, status=None, fill=7.0, stream=None):
    pages = yl.KvPages.of(k, v)
    batch = g.device(yl, status, shared)
    out = torch.full((g.n_rows, g.heads, g.hd), fill, dtype=out_dtype or q.dtype, device="cuda")
    lse = torch.full((g.n_rows, g.heads), fill, device="cuda")
    ws = torch.full((yl.paged_attention_workspace(pages, batch, g.heads),), 0xFF, dtype=torch.uint8, device="cuda")
    yl.paged_attention(out, q, pages, batch, g.heads, scale, ws, lse=lse, stream=stream)
    return out, lse


def queries(g, dtype, std=2.0):
    return torch.from_numpy(g.rng.standard_normal((g.n_rows, g.heads, g.hd)) * std).to(dtype)


def check_attention(yl, g, dtype, shared=None, out_dtype=None):
    q, (k, v), scale = queries(g, dtype), g.pool(dtype), g.hd**-0.5
    out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), scale, out_dtype, shared)
    want, wlse, ob, lb = ref.attention(g, q, k, v, scale)
    new = int(g.row_start[-1])
    assert (out[new:] == 7.0).all() and (lse[new:] == 7.0).all()
    o = out.dtype
    within(out[:new], want[:new], (ob + (want.abs() + ob) * ref.half_step(o) + 2.0**-25 * (o == torch.float16))[:new],
           "out")
    within(lse[:new], wlse[:new], lb[:new], "lse")


# decode: one row per sequence; lengths around pages, tiles and 0
DECODE = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1025]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("page", [8, 64, 256])
def test_decode(yl, torch_cuda, dtype, shape, page):
    g = ref.Geometry(4, *shape, page=page, lens=DECODE, rows=[1] * len(DECODE), pad_rows=2)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(9, 3, 64), (8, 2, 128), (14, 2, 64)])
def test_prompts(yl, torch_cuda, dtype, shape):
    """Chunks of prompts: whole ones, later chunks, one row, none, more rows than tokens (the first see no key)."""
    g = ref.Geometry(5, *shape, page=16, lens=[70, 150, 33, 5, 0, 200, 3], rows=[70, 41, 1, 0, 2, 130, 6], pad_rows=5)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(9, 3, 64), (32, 8, 128)])
@pytest.mark.parametrize("shared", [16, 272, 1024])
def test_shared_prefix_decode(yl, torch_cuda, own_pass, dtype, shape, shared):
    lens = [shared + n for n in (0, 1, 5, 16, 17, 64, 90, 200, 333)]
    g = ref.Geometry(6, *shape, page=16, lens=lens, rows=[1] * 8 + [0], shared=shared, pad_rows=1)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(9, 3, 64), (8, 2, 128)])
def test_shared_prefix_prompts(yl, torch_cuda, own_pass, dtype, shape):
    """Rows behind the prefix, and rows inside it (a sequence whose chunk begins before the prefix ends)."""
    g = ref.Geometry(7, *shape, page=32, lens=[96 + 70, 96 + 1, 100, 96], rows=[70, 1, 60, 96], shared=96)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype,kv,n", [("f32", 2, 3), ("f16", 2, 8), ("bf16", 1, 50), ("f16", 4, 40)])
def test_shared_prefix_where_it_pays(yl, torch_cuda, dtype, kv, n):
    """The rule's own choice: prefixes long enough for a pass of their own (passes side by side, and on tcgen05), and
    the same without one, which is held to the same bounds."""
    shared = 12288
    g = ref.Geometry(40, 4 * kv, kv, 64, page=64, lens=shared + np.arange(n) * 7, rows=[1] * n, shared=shared)
    batch = g.device(yl)
    k, v = (torch.empty(g.n_pages, 64, kv, 64, dtype=DTYPES[dtype], device="cuda") for _ in range(2))
    with_pass = yl.paged_attention_workspace(yl.KvPages.of(k, v), batch, g.heads)
    yl.config_set("paged_share", 0)
    try:
        without = yl.paged_attention_workspace(yl.KvPages.of(k, v), batch, g.heads)
        check_some_rows(yl, g, DTYPES[dtype], [0, n // 2, n - 1])
    finally:
        yl.config_set("paged_share", -1)
    assert with_pass > without
    check_some_rows(yl, g, DTYPES[dtype], [0, n // 2, n - 1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 64])
def test_f32_output_of_16_bit_cache(yl, torch_cuda, own_pass, dtype, shared):
    g = ref.Geometry(8, 8, 2, 128, page=32, lens=[64 + 30, 64 + 129, 65], rows=[1, 40, 1], shared=64)
    check_attention(yl, g, DTYPES[dtype], shared=shared, out_dtype=torch.float32)


def test_long_rows(yl, torch_cuda, own_pass):
    """Long sequences, split over many blocks: one token against 40000, next to short ones."""
    for dtype in ("f32", "bf16"):
        g = ref.Geometry(9, 2, 1, 64, page=64, lens=[40000, 3, 12345], rows=[1, 1, 2])
        check_attention(yl, g, DTYPES[dtype])
    g = ref.Geometry(9, 2, 1, 64, page=64, lens=[20480 + 3, 20480 + 3000], rows=[1, 2], shared=20480)
    check_attention(yl, g, torch.float16)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts(yl, torch_cuda, own_pass, dtype):
    """Heads before tokens, keys and values interleaved by page, one layer of several, q and output rows inside wider
    ones: the same bits as the plain layout."""
    t = DTYPES[dtype]
    g = ref.Geometry(10, 8, 2, 64, page=16, lens=[50, 130, 33], rows=[1, 20, 2], shared=32)
    q, (k, v) = queries(g, t).cuda(), (x.cuda() for x in g.pool(t))
    out, lse = attend(yl, g, q, k, v, 0.125)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    both = torch.stack([k, v], 1)
    layers = torch.zeros(g.n_pages, 3, 2, g.page, g.kv, g.hd, dtype=t, device="cuda")
    layers[:, 1, 0], layers[:, 1, 1] = k, v
    for a, b in (heads_first, (both[:, 0], both[:, 1]), (layers[:, 1, 0], layers[:, 1, 1])):
        assert a.stride() == b.stride()
        o2, l2 = attend(yl, g, q, a, b, 0.125)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
    pages, batch = yl.KvPages.of(k, v), g.device(yl)
    wide = torch.full((g.n_rows, g.heads * g.hd + 32), 7.0, dtype=t, device="cuda")
    qw = torch.cat([q.flatten(1), q.flatten(1)], 1)[:, : g.heads * g.hd]
    ws = torch.empty(yl.paged_attention_workspace(pages, batch, g.heads), dtype=torch.uint8, device="cuda")
    yl.paged_attention(wide[:, : g.heads * g.hd], qw, pages, batch, g.heads, 0.125, ws)
    assert torch.equal(wide[:, : g.heads * g.hd].reshape(out.shape), out) and (wide[:, g.heads * g.hd :] == 7.0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_garbage_behind_the_sequences(yl, torch_cuda, own_pass, dtype, bad):
    """Slots behind a sequence's last position and pages of nobody hold NaN or infinities: nothing changes."""
    t = DTYPES[dtype]
    g = ref.Geometry(11, 8, 2, 64, page=32, lens=[64 + 9, 64 + 70, 64, 67], rows=[1, 20, 1, 3], shared=64)
    q, (k, v) = queries(g, t).cuda(), g.pool(t)
    used = torch.zeros(g.n_pages, g.page, dtype=torch.bool)
    for i, n in enumerate(g.lens):
        for p in range(n):
            used[int(g.table[i, p // g.page]), p % g.page] = True
    for shared in (64, 0):
        clean = attend(yl, g, q, k.cuda(), v.cuda(), 0.125, shared=shared)
        dirty = [torch.where(used[..., None, None], x, torch.tensor(bad, dtype=t)).cuda() for x in (k, v)]
        got = attend(yl, g, q, *dirty, 0.125, shared=shared)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


def test_not_finite_keys_reach_their_readers_only(yl, torch_cuda):
    """NaN in one sequence's cache stays in that sequence."""
    for rows in ([1, 1, 1], [20, 30, 40]):
        g = ref.Geometry(12, 4, 2, 64, page=16, lens=[40, 50, 60], rows=rows)
        mine = slice(rows[0], rows[0] + rows[1])
        others = [i for i in range(sum(rows)) if i not in range(mine.start, mine.stop)]
        for t in DTYPES.values():
            for bits in (0x7FFFFFFF, 0x7FC00000, -1):  # all ones, as arithmetic makes it, and torch's, and a negative one
                q, (k, v) = queries(g, t).cuda(), (x.cuda() for x in g.pool(t))
                clean, _ = attend(yl, g, q, k, v, 0.125)
                ints = torch.int32 if t == torch.float32 else torch.int16
                k.view(ints)[int(g.table[1, 0]), 3] = bits if t == torch.float32 else (bits >> 16 if bits > 0 else -1)
                assert k[int(g.table[1, 0]), 3].isnan().all()
                got, lse = attend(yl, g, q, k, v, 0.125)
                assert torch.equal(got[others], clean[others]) and got[mine].isnan().all() and lse[mine].isnan().all()


def test_bad_pages_and_missing_slots(yl, torch_cuda):
    """Ids that are no pages read as zeros; keys behind the table's last slot are left out. The status word tells."""
    for t in DTYPES.values():
        for where in ("page", "slot"):
            g = ref.Geometry(13, 4, 2, 64, page=16, lens=[40, 130], rows=[1, 2], spare_slots=0)
            q, (k, v) = queries(g, t), g.pool(t)
            if where == "page":
                g.table[1, 3] = 0xFFFFFFF0
                want = ref.attention(g, q, k, v, 0.125)
            else:  # both rows of the second sequence see what six pages hold
                want = ref.attention(g, q, k, v, 0.125, limit=96)
                g.table = g.table[:, :6].copy()
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.125, status=status)
            assert status.item() == -6
            within(out, want[0], want[2] + (want[0].abs() + want[2]) * ref.half_step(t) + 2.0**-25 * (t == torch.float16), "out")
            within(lse, want[1], want[3], "lse")


def test_large_scores(yl, torch_cuda):
    """Scores of several hundred, both signs: the running maximum keeps exp in range."""
    for t in DTYPES.values():
        g = ref.Geometry(14, 4, 1, 64, page=16, lens=[200, 90], rows=[2, 70])
        q, (k, v) = queries(g, t, 40.0), g.pool(t)
        out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.5)
        want, wlse, ob, lb = ref.attention(g, q, k, v, 0.5)
        within(out, want, ob + (want.abs() + ob) * ref.half_step(t) + 2.0**-25 * (t == torch.float16), "out")
        within(lse, wlse, lb, "lse")


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales(yl, torch_cuda, scale):
    """A negative scale, and one of 0 (every visible key alike)."""
    for t in DTYPES.values():
        g = ref.Geometry(20, 4, 1, 64, page=16, lens=[200, 90, 0], rows=[1, 70, 1])
        q, (k, v) = queries(g, t), g.pool(t)
        out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), scale)
        want, wlse, ob, lb = ref.attention(g, q, k, v, scale)
        within(out, want, ob + (want.abs() + ob) * ref.half_step(t) + 2.0**-25 * (t == torch.float16), "out")
        within(lse, wlse, lb, "lse")


def test_cache_beyond_32_bits(yl, torch_cuda):
    """Pages whose elements lie beyond 2^32 (a view with a large page stride over one allocation)."""
    hd, kv, page = 64, 1, 8
    n_pages, stride = 5, 1 << 30
    big = torch.empty(4 * stride + 2 * page * kv * hd, dtype=torch.float16, device="cuda")
    k = big.as_strided((n_pages, page, kv, hd), (stride, kv * hd, hd, 1))
    v = big[page * kv * hd :].as_strided((n_pages, page, kv, hd), (stride, kv * hd, hd, 1))
    g = ref.Geometry(15, 2, kv, hd, page=page, lens=[40], rows=[1], spare_pages=0)
    q, (kh, vh) = queries(g, torch.float16), g.pool(torch.float16)
    k.copy_(kh), v.copy_(vh)
    out, lse = attend(yl, g, q.cuda(), k, v, 0.125)
    want, wlse, ob, lb = ref.attention(g, q, kh, vh, 0.125)
    within(out, want, ob + (want.abs() + ob) * ref.half_step(torch.float16) + 2.0**-25, "out")
    within(lse, wlse, lb, "lse")


def test_same_bits_again_and_on_another_stream(yl, torch_cuda, own_pass):
    g = ref.Geometry(16, 8, 2, 128, page=16, lens=[512 + 900, 512 + 3, 512 + 77], rows=[1, 1, 1], shared=512)
    q, (k, v) = queries(g, torch.bfloat16).cuda(), (x.cuda() for x in g.pool(torch.bfloat16))
    first = attend(yl, g, q, k, v, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            again = attend(yl, g, q, k, v, 0.1)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    torch.cuda.current_stream().wait_stream(side)


def check_some_rows(yl, g, dtype, rows, shared=None):
    q, (k, v), scale = queries(g, dtype), g.pool(dtype), g.hd**-0.5
    out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), scale, shared=shared)
    only = set(int(r) for r in rows)
    want, wlse, ob, lb = ref.attention(g, q, k, v, scale, only=only)
    at = sorted(only)
    within(out[at], want[at], (ob + (want.abs() + ob) * ref.half_step(dtype) + 2.0**-25 * (dtype == torch.float16))[at], "out")
    within(lse[at], wlse[at], lb[at], "lse")
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_one_long_prompt(yl, torch_cuda, dtype):
    """More row tiles than a warp counts at a time, key tiles cut among all blocks; rows next to tile borders."""
    n = 5003
    g = ref.Geometry(30, 2, 1, 64, page=32, lens=[n], rows=[n])
    rows = [0, 1, 31, 32, 63, 64, 127, 128, 129, 255, 256, n - 130, n - 129, n - 2, n - 1] + list(
        np.random.default_rng(0).integers(0, n, 40))
    check_some_rows(yl, g, DTYPES[dtype], rows)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_many_sequences(yl, torch_cuda, own_pass, dtype):
    """More sequences than a block has threads, idle slots among them."""
    rng = np.random.default_rng(31)
    lens = rng.integers(1, 90, 700)
    rows = (rng.random(700) < 0.8).astype(int)
    g = ref.Geometry(31, 2, 1, 64, page=16, lens=lens, rows=rows, pad_rows=9)
    check_some_rows(yl, g, DTYPES[dtype], rng.integers(0, int(g.row_start[-1]), 120))
    lens, rows = lens + 64, rng.integers(0, 4, 700)
    g = ref.Geometry(32, 4, 2, 64, page=16, lens=lens, rows=rows, shared=64)
    check_some_rows(yl, g, DTYPES[dtype], rng.integers(0, int(g.row_start[-1]), 120))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_mixed_prompts_and_tokens(yl, torch_cuda, own_pass, dtype):
    """One prompt chunk next to single tokens, with and without a shared prefix."""
    for shared in (0, 128):
        g = ref.Geometry(33, 6, 2, 128, page=64, lens=[shared + n for n in (400, 1, 17, 90, 300)], rows=[300, 1, 1, 1, 2],
                         shared=shared)
        check_some_rows(yl, g, DTYPES[dtype], np.random.default_rng(1).integers(0, 305, 60))


@pytest.mark.parametrize("seed", range(24))
def test_random_geometries(yl, torch_cuda, own_pass, seed):
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *a: a[rng.integers(len(a))]  # noqa: E731
    kv, group, hd = pick(1, 2, 3), pick(1, 2, 3, 4, 5, 7, 8, 12, 16), pick(64, 128)
    page, n = pick(8, 16, 32, 64, 128, 256), int(rng.integers(1, 9))
    shared = pick(0, 0, 1, 2, 5) * page
    lens = shared + np.array([pick(0, 1, 7, 64, 65, int(rng.integers(1, 400))) for _ in range(n)])
    rows = [min(int(x) + 2, pick(0, 1, 1, 3, 17, int(rng.integers(1, 100)))) for x in lens]
    g = ref.Geometry(seed, kv * group, kv, hd, page=page, lens=lens, rows=rows, shared=shared, pad_rows=pick(0, 3))
    if not g.n_rows:
        return
    check_attention(yl, g, pick(*DTYPES.values()), shared=pick(0, shared))


def test_row_starts_behind_zero_and_out_of_order(yl, torch_cuda):
    """Rows before row_start[0] belong to nobody. Starts beyond n_rows or that run backwards stay within the rows."""
    g = ref.Geometry(34, 4, 2, 64, page=16, lens=[30, 60, 40], rows=[2, 1, 3])
    for t in DTYPES.values():
        (k, v) = (x.cuda() for x in g.pool(t))
        q = queries(g, t)
        want, _ = attend(yl, g, q.cuda(), k, v, 0.125)
        shifted = ref.Geometry(34, 4, 2, 64, page=16, lens=[30, 60, 40], rows=[2, 1, 3], pad_rows=4)
        shifted.table, shifted.row_start = g.table, g.row_start + 4
        qs = torch.cat([torch.zeros(4, 4, 64, dtype=t), q])
        got, lse = attend(yl, shifted, qs.cuda(), k, v, 0.125)
        assert torch.equal(got[4:], want) and (got[:4] == 7.0).all() and (lse[:4] == 7.0).all()
        for starts in ([0, 5, 2, 6], [9, 9, 9, 9], [0, 2, 100, 0xFFFFFFF0], [6, 4, 2, 0]):
            shifted.row_start = np.array(starts, np.uint32)
            attend(yl, shifted, qs.cuda(), k, v, 0.125)
            yl.paged_append(torch.zeros(10, 8 * 64, device="cuda"), yl.KvPages.of(k.clone(), v.clone()), shifted.device(yl), 4)
    torch.cuda.synchronize()


def test_captured_step_follows_its_arrays(yl, torch_cuda, own_pass):
    """Append, attention and log probabilities captured once and replayed while the sequences grow: the arrays' new
    contents count, and each replay equals the eager calls."""
    t, hd, heads, kv, vocab = torch.bfloat16, 64, 8, 2, 5000
    n, page, slots, shared = 5, 16, 12, 32
    rng = np.random.default_rng(5)
    table = np.concatenate([np.tile([0, 1], (n, 1)), 2 + rng.permutation(n * (slots - 2)).reshape(n, -1)], 1)
    arrays = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (np.arange(n + 1), np.full(n, 40), table)]
    pools = [torch.randn(2 + n * (slots - 2), page, kv, hd, device="cuda").to(t) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = yl.SeqBatch(*arrays, n, shared_len=shared, status=status)
    cs = ref.rope_cs(slots * page, hd).cuda()
    qkv, logits = torch.empty(n, (heads + 2 * kv) * hd, device="cuda"), torch.empty(n, vocab, device="cuda")
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")

    def buffers():
        return dict(q=torch.empty(n, heads, hd, dtype=t, device="cuda"), out=torch.empty(n, heads, hd, dtype=t, device="cuda"),
                    lse=torch.empty(n, heads, device="cuda"), lp=torch.empty(n, device="cuda"),
                    ids=torch.empty(n, 4, dtype=torch.int32, device="cuda"), top=torch.empty(n, 4, device="cuda"))

    def step(pages, b, ws):
        yl.paged_append(qkv, pages, batch, heads, rope_cs=cs, q_out=b["q"])
        yl.paged_attention(b["out"], b["q"], pages, batch, heads, 0.125, ws, lse=b["lse"])
        yl.token_logprobs(logits, tokens, b["lp"], top_ids=b["ids"], top_logprobs=b["top"])

    pages = yl.KvPages.of(*pools)
    size = yl.paged_attention_workspace(pages, batch, heads)
    ws, ws2 = (torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    a, b = buffers(), buffers()
    qkv.normal_(), logits.normal_()
    step(pages, a, ws)  # (loads the kernels)
    twin_pages = yl.KvPages.of(*[x.clone() for x in pools])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pages, a, ws)
    for i in range(6):
        arrays[1].copy_(torch.tensor([33 + i, 40 + 20 * i, 60 + i, 33, 160 + i], dtype=torch.int32))
        qkv.normal_(), logits.normal_()
        graph.replay()
        step(twin_pages, b, ws2)
        for name in a:
            assert torch.equal(a[name], b[name]), (i, name)
    assert status.item() == 0
    arrays[1][4] = 1000  # beyond the table
    graph.replay()
    assert status.item() == -6


def test_two_calls_at_once(yl, torch_cuda):
    """Two streams, a workspace each."""
    g = ref.Geometry(35, 8, 2, 128, page=16, lens=[900, 3000, 50, 2000], rows=[1, 1, 1, 1])
    h = ref.Geometry(36, 8, 2, 128, page=16, lens=[900, 700], rows=[300, 500])
    ops = []
    for x in (g, h):
        q, (k, v) = queries(x, torch.float16).cuda(), (y.cuda() for y in x.pool(torch.float16))
        ops.append((x, q, k, v, attend(yl, x, q, k, v, 0.1)[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    got = [[], []]
    for _ in range(10):
        for i, (s, (x, q, k, v, _)) in enumerate(zip(streams, ops)):
            with torch.cuda.stream(s):
                got[i].append(attend(yl, x, q, k, v, 0.1)[0])
    torch.cuda.synchronize()
    for i, (_, _, _, _, want) in enumerate(ops):
        assert all(torch.equal(o, want) for o in got[i])


def test_python_refusals(yl, torch_cuda):
    g = ref.Geometry(37, 4, 2, 64, page=16, lens=[30], rows=[2])
    k, v = (x.cuda() for x in g.pool(torch.float16))
    pages, batch = yl.KvPages.of(k, v), g.device(yl)
    q, out = (torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    ws = torch.empty(yl.paged_attention_workspace(pages, batch, 4), dtype=torch.uint8, device="cuda")
    qkv = torch.zeros(2, 8 * 64, device="cuda")
    lp = torch.zeros(2, device="cuda")
    attend_ = lambda **kw: yl.paged_attention(**{**dict(output=out, q=q, pages=pages, batch=batch, n_heads=4,  # noqa: E731
                                                       attn_scale=0.1, workspace=ws), **kw})
    append_ = lambda **kw: yl.paged_append(**{**dict(qkv=qkv, pages=pages, batch=batch, n_heads=4), **kw})  # noqa: E731
    for kind, call in (
            (TypeError, lambda: attend_(q=q.float())), (TypeError, lambda: attend_(output=out.double())),
            (yl.YlError, lambda: attend_(output=out.bfloat16())), (ValueError, lambda: attend_(q=q[:1])),
            (ValueError, lambda: attend_(q=q.cpu())), (ValueError, lambda: attend_(q=q.transpose(1, 2))),
            (yl.YlError, lambda: attend_(workspace=ws[: ws.numel() // 2])), (TypeError, lambda: attend_(workspace=ws.float())),
            (ValueError, lambda: attend_(lse=lp)), (ValueError, lambda: attend_(n_heads=8)),
            (TypeError, lambda: append_(qkv=qkv.half())), (ValueError, lambda: append_(qkv=qkv[:, 1:])),
            (TypeError, lambda: append_(q_out=q.float())), (ValueError, lambda: append_(rope_cs=lp)),
            (ValueError, lambda: yl.KvPages.of(k, v[:, :8])), (ValueError, lambda: yl.KvPages.of(k.cpu(), v.cpu())),
            (ValueError, lambda: yl.SeqBatch(batch._keep[0], batch._keep[1], batch._keep[2][0], 2)),
            (TypeError, lambda: yl.SeqBatch(batch._keep[0].long(), batch._keep[1], batch._keep[2], 2)),
            (TypeError, lambda: yl.token_logprobs(qkv.double(), entropy=lp)),
            (TypeError, lambda: yl.token_logprobs(qkv, lp, lp)), (ValueError, lambda: yl.token_logprobs(qkv.t(), entropy=lp)),
            (yl.YlError, lambda: yl.token_logprobs(qkv, logprobs=lp))):
        with pytest.raises(kind):
            call()
    attend_(), append_()


def test_pages_from_the_library(yl, torch_cuda):
    """A cache that the library allocates: append, then attend, as with torch's."""
    g = ref.Geometry(38, 4, 2, 64, page=16, lens=[5], rows=[5])
    qkv = torch.from_numpy(g.rng.standard_normal((5, 8 * 64))).float().cuda()
    k, v = torch.zeros(g.n_pages, 16, 2, 64, device="cuda"), torch.zeros(g.n_pages, 16, 2, 64, device="cuda")
    mine = yl.KvPages.alloc(yl.DType.F32, g.n_pages, 16, 2, 64)
    batch, outs = g.device(yl), []
    for pages in (yl.KvPages.of(k, v), mine):
        q, out = torch.empty(5, 4, 64, device="cuda"), torch.empty(5, 4, 64, device="cuda")
        yl.paged_append(qkv, pages, batch, 4, q_out=q)
        ws = torch.empty(yl.paged_attention_workspace(pages, batch, 4), dtype=torch.uint8, device="cuda")
        yl.paged_attention(out, q, pages, batch, 4, 0.125, ws)
        outs.append(out)
    assert torch.equal(*outs)
    torch.cuda.synchronize()
    mine.free()


@pytest.mark.parametrize("preset,over", [("tiny", {}), ("tiny", {"llama3_scaling": True}), ("tiny128", {})])
def test_a_model_layer_served_from_pages(yl, torch_cuda, own_pass, model_factory, preset, over):
    """The step of a server, next to the library's own: the projections of a model's first layer on the rows of three
    sequences that share a prefix, the rows appended with the model's rotation table, attention over the pages. Keys and
    values in an f32 cache have the bits of the decode kernel's cache, the outputs agree within the f32 bound, and a
    bf16 cache within its own."""
    m = yl.load_transformer(model_factory(preset, **over), max_ctx_len=256)
    sh = m.shape()
    heads, kv, hd, dim = sh.n_heads, sh.n_kv_heads, sh.head_size, sh.dim
    cs, cs_len = m.rope_table()
    mode = yl.ROPE_LLAMA3 if sh.rope_mode else yl.ROPE_GGUF
    scale = 1.0 / math.sqrt(hd)
    lens, shared, page = [70, 41, 33], 32, 16

    def project(x):
        act = yl.new_workspace_buffer(yl.WeightFormat.Q8_0, x.numel(), 32)
        yl.quantize(yl.WeightFormat.Q8_0, act, x, x.numel(), 32)
        parts = []
        for which, rows in ((0, heads * hd), (1, kv * hd), (2, kv * hd)):
            out = torch.zeros(x.shape[0], rows, device="cuda")
            yl.matmul(out, act, m.weight(0, which), dim, rows, 32, accumulate=False)
            parts.append(out)
        return torch.cat(parts, 1)

    gen = torch.Generator(device="cuda").manual_seed(3)
    prefix = torch.randn(shared, dim, generator=gen, device="cuda") * 4
    own = [torch.randn(n - shared, dim, generator=gen, device="cuda") * 4 for n in lens]
    qkv_prefix, qkv_own = project(prefix), [project(x) for x in own]
    for dtype in (torch.float32, torch.bfloat16):
        g = ref.Geometry(39, heads, kv, hd, page=page, lens=lens, rows=[1, 1, 1], shared=shared)
        k, v = (torch.zeros(g.n_pages, page, kv, hd, dtype=dtype, device="cuda") for _ in range(2))
        pages = yl.KvPages.of(k, v)

        def append(rows, counts, upto, q_out=None):
            part = ref.Geometry(39, heads, kv, hd, page=page, lens=upto, rows=counts, shared=shared)
            part.table = g.table[: len(upto)]
            yl.paged_append(rows, pages, part.device(yl), heads, rope_cs=cs, rope_len=cs_len, rope_mode=mode, q_out=q_out)

        append(qkv_prefix, [shared], [shared])  # the prefix once, through the first sequence's table
        append(torch.cat([x[:-1] for x in qkv_own]), [n - shared - 1 for n in lens], [n - 1 for n in lens])
        last = torch.cat([x[-1:] for x in qkv_own])
        q, out = (torch.empty(3, heads, hd, dtype=dtype, device="cuda") for _ in range(2))
        append(last, [1, 1, 1], lens, q)
        batch = g.device(yl)
        ws = torch.empty(yl.paged_attention_workspace(pages, batch, heads), dtype=torch.uint8, device="cuda")
        yl.paged_attention(out, q, pages, batch, heads, scale, ws)
        want, _, ob, _ = ref.attention(g, q.cpu(), k.cpu(), v.cpu(), scale)
        within(out, want, ob + (want.abs() + ob) * ref.half_step(dtype), "out")
        if dtype != torch.float32:
            continue
        for i, n in enumerate(lens):  # the decode kernel on a cache of its own
            kc, vc, o = (torch.zeros(n, kv * hd, device="cuda") for _ in range(3))
            o = torch.zeros(heads * hd, device="cuda")
            for pos, row in enumerate(torch.cat([qkv_prefix, qkv_own[i]])):
                m.attention_decode(row.contiguous(), kc, vc, pos, out=o)
            assert torch.equal(g.gather(i, k.cpu()), kc.cpu().double().view(n, kv, hd))
            assert torch.equal(g.gather(i, v.cpu()), vc.cpu().double().view(n, kv, hd))
            bound = 2 * ob[i].flatten() + 2 * want[i].abs().flatten() * ref.U32
            within(out[i].flatten(), o.double().cpu(), bound, "decode kernel")
    m.close()


def test_logprobs_of_sessions_and_batches(yl, torch_cuda, model_factory):
    """Log probabilities straight from the device logits of a session and of a batch, against the host's logits."""
    m = yl.load_transformer(model_factory("tiny"), max_ctx_len=64)
    vocab = m.vocab_size()
    sessions = [m.create_session() for _ in range(3)]
    for i, s in enumerate(sessions):
        logits, best = m.forward_x_full([1 + i, 7, 9], 0, s)
        lp, ids, top = torch.empty(1, device="cuda"), torch.empty(1, 3, dtype=torch.int32, device="cuda"), torch.empty(1, 3, device="cuda")
        yl.token_logprobs(yl.session_logits(s), torch.tensor([best], dtype=torch.int32, device="cuda"), lp, top_ids=ids,
                          top_logprobs=top, shape=(1, vocab))
        want = ref.logprobs(torch.from_numpy(logits)[None], torch.tensor([best]), 3)
        within(lp, want[0], want[4], "lp")
        assert ids.tolist() == want[2].tolist() and ids[0, 0].item() == best
    b = m.create_batch(3)
    _, logits = b.forward(sessions, [5, 6, 7], [3, 3, 3], want_logits=True)
    tokens = torch.tensor([1, 2, 3], dtype=torch.int32)
    lp, en = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    yl.token_logprobs(b.logits(), tokens.cuda(), lp, entropy=en, shape=(3, vocab))
    want = ref.logprobs(torch.from_numpy(logits), tokens, 0)
    within(lp, want[0], want[4], "lp")
    within(en, want[1], want[5], "entropy")
    b.close()
    for s in sessions:
        s.close()
    m.close()


# -------------------------------------------------------------- logprobs ---

def run_logprobs(yl, x, tokens, k):
    n = x.shape[0]
    lp, en = torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    ids = torch.full((n, k), 7, dtype=torch.int32, device="cuda")
    top = torch.full((n, k), 7.0, device="cuda")
    yl.token_logprobs(x, tokens, lp, entropy=en, top_ids=ids if k else None, top_logprobs=top if k else None)
    return lp.cpu(), en.cpu(), ids.cpu(), top.cpu()


def check_logprobs(yl, x, tokens, k, device_x=None):
    lp, en, ids, top = run_logprobs(yl, x.cuda() if device_x is None else device_x, tokens.cuda(), k)
    want = ref.logprobs(x, tokens, k)
    assert np.array_equal(ids.numpy(), want[2])
    within(lp, want[0], want[4], "logprobs")
    within(en, want[1], want[5], "entropy")
    within(top, want[3], want[6], "top_logprobs")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4097, 49152, 128256])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_logprobs(yl, torch_cuda, dtype, vocab, rows):
    if rows * vocab > 10_000_000:
        rows = 40
    rng = np.random.default_rng(vocab + rows)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * 4).to(DTYPES[dtype])
    tokens = torch.from_numpy(rng.integers(0, vocab, rows).astype(np.int32))
    tokens[0] = int(x[0].float().argmax())
    for k in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        check_logprobs(yl, x, tokens, k)


def test_logprobs_ties_and_masks(yl, torch_cuda):
    """Few distinct values, so that the order among equals decides; masks of -inf and of the type's lowest value;
    fewer unmasked tokens than alternatives; zeros of both signs."""
    rng = np.random.default_rng(0)
    for name, t in DTYPES.items():
        for vocab in (40, 5000, 70000):
            x = torch.from_numpy(rng.integers(-3, 3, (4, vocab)).astype(np.float64)).to(t)
            x[1, rng.random(vocab) < 0.9] = -math.inf
            x[2] = -math.inf
            x[2, 7], x[2, vocab - 1] = 1.0, 1.5
            x[3] = torch.finfo(t).min
            x[3, 11:20] = 2.0
            tokens = torch.tensor([5, int(x[1].float().argmax()), 7, 0], dtype=torch.int32)
            check_logprobs(yl, x, tokens, 20)
            z = torch.zeros(2, vocab, dtype=t)
            z[0, 1::3] = -0.0
            z[1] = torch.finfo(t).min  # nothing but the lowest value: every token alike
            check_logprobs(yl, z, torch.tensor([1, 2], dtype=torch.int32), 32)


def test_logprobs_many_large_values_in_one_place(yl, torch_cuda):
    """Large values that one thread reads all of (a stride apart), or that lie together, and sorted rows."""
    vocab = 128256
    for t in DTYPES.values():
        x = torch.from_numpy(np.random.default_rng(1).standard_normal((5, vocab))).to(t)
        x[0, :: 512 * (16 // t.itemsize)] += 50
        for j in range(40):
            x[1, j :: 512 * (16 // t.itemsize)] += 50
        x[2, 60000:60100] += 50
        x[3] = x[3].sort()[0]
        x[4] = x[4].sort(descending=True)[0]
        check_logprobs(yl, x, torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32), 32)
    x = torch.randn(300, 16000)  # one block a row
    x[:, :: 2048] += 60
    for j in range(32):
        x[7, j :: 2048] += 60
    x[8] = x[8].sort()[0]
    check_logprobs(yl, x, torch.arange(300, dtype=torch.int32), 32)


def test_logprobs_near_certain(yl, torch_cuda):
    """A token of probability 1 - 1e-9: its log probability and the entropy keep their digits."""
    x = torch.zeros(2, 1000)
    x[0, 10], x[1, 999] = 27.0, 60.0
    lp, en, ids, top = run_logprobs(yl, x.cuda(), torch.tensor([10, 999], dtype=torch.int32).cuda(), 2)
    for i, m in enumerate((27.0, 60.0)):
        s = 999 * math.exp(-m)
        # sums of 999 equal terms and their exp: 100 half steps; 27 and 60 in f32 times log2(e): |d| * 4
        rel = (100 + 4 * m) * ref.U32
        assert abs(lp[i].item() + math.log1p(s)) <= rel * s
        assert abs(en[i].item() - (math.log1p(s) + s * m / (1 + s))) <= 2 * rel * s * m
        assert ids[i].tolist() == [[10, 0], [999, 0]][i]


def test_logprobs_rows_without_a_distribution(yl, torch_cuda):
    for vocab in (100, 50000):
        x = torch.randn(6, vocab)
        x[0, 3], x[1, vocab - 1], x[2], x[3, 5:7] = math.nan, math.inf, -math.inf, math.inf
        x[4] = math.nan
        lp, en, ids, top = run_logprobs(yl, x.cuda(), torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32).cuda(), 3)
        assert lp[:5].isnan().all() and en[:5].isnan().all() and top[:5].isnan().all() and (ids[:5] == -1).all()
        assert lp[5].isfinite() and en[5].isfinite() and (ids[5] >= 0).all()
        lp, en, _, _ = run_logprobs(yl, x[5:].cuda(), torch.tensor([vocab], dtype=torch.int32).cuda(), 0)
        assert lp.isnan().all() and en.isfinite().all()
        lp, en, _, _ = run_logprobs(yl, x[5:].cuda(), torch.tensor([-1], dtype=torch.int32).cuda(), 0)
        assert lp.isnan().all() and en.isfinite().all()


def test_logprobs_rows_inside_wider_ones(yl, torch_cuda):
    """Odd strides and starts: rows not aligned to 16 bytes."""
    for t in DTYPES.values():
        for start, vocab, stride in ((1, 4999, 5003), (3, 997, 1001), (2, 30001, 30011)):
            wide = torch.randn(5, stride + 8).to(t)
            dev = wide.cuda()
            x = wide[:, start : start + vocab].contiguous()
            check_logprobs(yl, x, torch.tensor([0, 1, vocab - 1, 3, 4], dtype=torch.int32), 7,
                           device_x=dev[:, start : start + vocab])


# ------------------------------------------------------------ the mirror ---

def test_calls_without_rows(yl, torch_cuda):
    """Tensors of no rows have no address; the calls return and touch nothing."""
    g = ref.Geometry(50, 8, 2, 64, page=16, lens=[20, 5], rows=[0, 0])
    k, v = (x.cuda() for x in g.pool(torch.bfloat16))
    before, pages, batch = k.clone(), yl.KvPages.of(k, v), g.device(yl)
    assert batch.n_rows == 0
    q = torch.empty(0, 8, 64, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(yl.paged_attention_workspace(pages, batch, 8), dtype=torch.uint8, device="cuda")
    yl.paged_append(torch.empty(0, 12 * 64, device="cuda"), pages, batch, 8, q_out=q)
    yl.paged_attention(torch.empty_like(q), q, pages, batch, 8, 0.1, ws)
    i32, f32 = (torch.empty(0, 4, dtype=t, device="cuda") for t in (torch.int32, torch.float32))
    yl.token_logprobs(torch.empty(0, 100, device="cuda"), i32[:, 0], f32[:, 0], f32[:, 0], i32, f32)
    torch.cuda.synchronize()
    assert torch.equal(k, before)


def test_mirror_refusals(yl, torch_cuda):
    """Cache or batch of another device than the current one, halves of the alternatives' outputs, alternatives of
    different shapes."""
    g = ref.Geometry(51, 8, 2, 64, page=16, lens=[20, 5], rows=[1, 1])
    k, v = (x.cuda() for x in g.pool(torch.float32))
    q, qkv = torch.zeros(2, 8, 64, device="cuda"), torch.zeros(2, 12 * 64, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    for which in ("pages", "batch"):
        pages, batch = yl.KvPages.of(k, v), g.device(yl)
        (pages if which == "pages" else batch).device += 1
        with pytest.raises(ValueError):
            yl.paged_append(qkv, pages, batch, 8)
        with pytest.raises(ValueError):
            yl.paged_attention(q.clone(), q, pages, batch, 8, 0.1, ws)
    x = torch.zeros(3, 50, device="cuda")
    ids, lp = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, device="cuda")
    for a, b in ((ids, None), (None, lp), (ids, torch.zeros(3, 5, device="cuda"))):
        with pytest.raises(ValueError):
            yl.token_logprobs(x, top_ids=a, top_logprobs=b)


@pytest.mark.parametrize("dtype,rows", [("f32", 1), ("f32", 30), ("bf16", 1), ("bf16", 6), ("bf16", 90)])
def test_scores_beyond_f32(yl, torch_cuda, dtype, rows):
    """A finite score that overflows once it is scaled: NaN, not a row of zeros. Rows of other sequences are as ever."""
    t = DTYPES[dtype]
    g = ref.Geometry(52, 4, 1, 64, page=16, lens=[rows, 40], rows=[rows, rows if rows <= 40 else 40])
    q, (k, v) = queries(g, t), g.pool(t)
    q[:rows] = 1.5e18
    for p in g.positions(0):
        k[int(g.table[0, p // g.page]), int(p % g.page)] = 1.5e18
    out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 4.0)  # 64 * 2.25e36 * 4 log2(e) = 8.3e38
    assert out[:rows].isnan().all() and lse[:rows].isnan().all()
    assert out[rows:].isfinite().all() and lse[rows:].isfinite().all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [49152, 128256, 50001])
@pytest.mark.parametrize("rows", [1, 3, 64, 200])
def test_logprobs_near_certain_rows_of_several_blocks(yl, torch_cuda, dtype, vocab, rows):
    """Rows of one to eight blocks, nearly certain of a token anywhere in them (first and last values, odd rows of an odd
    vocabulary that begin and end inside 16 bytes): S' = S - 1 from 1e-9 over values a few last bits of 1 around the
    border 2^-7, where the sum is taken again, to 2^-5.
    Below the border everything is relative to S' (sums in chains of V/512 + 64 of two half steps each, exp of an f32
    difference d: |d| * 4 half steps, exp itself 8), above it S has lost what the general bound allows."""
    t = DTYPES[dtype]
    rng = np.random.default_rng(vocab + rows)
    gen = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = torch.randn(rows, vocab, generator=gen, device="cuda").to(t)
    places = [0, vocab - 1, vocab // 2, 1, vocab // 8, vocab // 8 - 1, vocab - 2, 7 * vocab // 8, 3, vocab // 4 + 1]
    at = torch.tensor([places[i % 10] if i < 20 else int(rng.integers(vocab)) for i in range(rows)], device="cuda")
    near = [2.0**-7 * (1 + (i % 17 - 8) * 2.0**-17) for i in range(rows)]
    target = torch.tensor([near[i] if i % 2 else (1e-9, 1e-6, 2.0**-12, 2.0**-8, 2.0**-6, 2.0**-5)[i // 2 % 6]
                           for i in range(rows)], dtype=torch.float64, device="cuda")
    r = torch.arange(rows, device="cuda")
    x[r, at] = -math.inf
    rest = x.double().exp().sum(1)
    x[r, at] = (rest / target).log().to(t)
    d = x.double() - x.double()[r, at][:, None]
    assert (d <= 0).all()
    e = d.exp()
    e[r, at] = 0.0
    s, w = e.sum(1), (e * d).sum(1)  # S', W
    far = float(-d.min())
    lp, en, ids, _ = run_logprobs(yl, x, at.int(), 2)
    rel = (vocab / 512 + 64) * 2 * ref.U32 + 8 * ref.U32 + 4 * ref.U32 * far
    below = s < 2.0**-7 * (1 - 2.0**-10)
    scale = torch.where(below, s, 1.0)
    within(lp, -s.log1p(), rel * scale + 4 * ref.U32 * s, "logprobs")
    within(en, s.log1p() - w / (1 + s), 2 * rel * scale * (1 + far) + 4 * ref.U32 * s * (1 + far), "entropy")
    assert torch.equal(ids[:, 0], at.cpu().int())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hd", [64, 128])
def test_hidden_values_weigh_nothing(yl, torch_cuda, own_pass, dtype, hd):
    """The last tokens' values are as large as the type allows, nearly: rows before them keep their bits, in chunks on
    tcgen05 and on mma.sync, and rows that end inside a shared prefix."""
    t = DTYPES[dtype]
    large = 6e4 if dtype == "f16" else 1e37
    for lens, rows, shared in (([100, 300], [100, 90], 0), ([40, 90, 33], [3, 4, 2], 0), ([128 + 40, 90], [30, 20], 128)):
        g = ref.Geometry(60, 4, 2, hd, page=32, lens=lens, rows=rows, shared=shared)
        q, (k, v) = queries(g, t), g.pool(t)
        clean = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.125)
        before = []
        for i, n in enumerate(lens):
            last = n - 20 if rows[i] > 20 else n - 1
            if shared and n < shared:
                continue  # (its last tokens are everyone's)
            for p in range(last, n):
                v[int(g.table[i, p // g.page]), p % g.page] = large
            before += [int(g.row_start[i]) + j for j, p in enumerate(g.positions(i)) if p < last]
        got = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.125)
        assert before and torch.equal(got[0][before], clean[0][before]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_garbage_in_a_prefix_behind_sequences_inside_it(yl, torch_cuda, own_pass, dtype, bad, hd):
    """Sequences that end inside the shared prefix do not see what lies behind them there: not a value that others read,
    nor what nobody has written yet. Decoding, small and large chunks, passes of every shape."""
    t = DTYPES[dtype]
    for lens, rows in (([100, 296, 257, 30, 326], [1, 1, 1, 1, 1]), ([100, 296, 257, 30, 326], [1, 3, 1, 3, 20]),
                       ([100, 30, 150], [1, 1, 1]), ([150, 30, 199], [30, 12, 20]),
                       ([100 + 3 * i for i in range(20)] + [270] * 20, [1] * 40)):
        g = ref.Geometry(61, 4, 2, hd, page=32, lens=lens, rows=rows, shared=256)
        q, (k, v) = queries(g, t), g.pool(t)
        check = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.125)
        want, wlse, ob, lb = ref.attention(g, q, k, v, 0.125)
        within(check[0], want, ob + (want.abs() + ob) * ref.half_step(t) + 2.0**-25 * (t == torch.float16), "out")
        within(check[1], wlse, lb, "lse")
        for p in range(200, 256):
            k[int(g.table[0, p // g.page]), p % g.page] = bad
            v[int(g.table[0, p // g.page]), p % g.page] = bad
        out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 0.125)
        for i, n in enumerate(lens):
            mine = slice(int(g.row_start[i]), int(g.row_start[i + 1]))
            if n <= 200:
                assert torch.equal(out[mine], check[0][mine]) and torch.equal(lse[mine], check[1][mine]), (lens, i)
            else:
                assert not out[mine].isfinite().any(), (lens, i)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 6, 30, 90])
def test_scores_below_f32(yl, torch_cuda, own_pass, dtype, rows):
    """Finite scores that overflow downwards once they are scaled: next to a score in range such a key weighs nothing,
    and a row of nothing else is NaN, not a row of zeros that looks like one without keys. In one piece, in many, and
    in passes that join."""
    t = DTYPES[dtype]
    for lens, shared in (([90, 100, 95], 0), ([5000, 90, 300], 0), ([64 + 90, 64 + 95, 64 + 100], 64)):
        n = min(rows, 30) if shared else rows
        g = ref.Geometry(62, 4, 1, 64, page=16, lens=lens, rows=[n, n, n], shared=shared)
        q, (k, v) = queries(g, t), g.pool(t)
        q[: 2 * n] = 1.5e18
        for i in (0, 1):
            for p in range(lens[i]):
                k[int(g.table[i, p // g.page]), p % g.page] = -1.5e18  # 64 * 2.25e36 * 4 log2(e) = 8.3e38
        k[int(g.table[1, (lens[1] - n) // g.page]), (lens[1] - n) % g.page] = 0.0  # every row's one key in range
        out, lse = attend(yl, g, q.cuda(), k.cuda(), v.cuda(), 4.0)
        assert out[:n].isnan().all() and lse[:n].isnan().all(), (lens, shared)
        one = v[int(g.table[1, (lens[1] - n) // g.page]), (lens[1] - n) % g.page].double()
        within(out[n : 2 * n], one.expand(n, 4, 64), (one.abs() * (2.0**-20 + ref.half_step(t))).expand(n, 4, 64), "one key")
        within(lse[n : 2 * n], torch.zeros(n, 4), torch.full((n, 4), 2.0**-20), "lse")
        if not shared:  # (the prefix's keys of the third are the others')
            want, wlse, ob, lb = ref.attention(g, q, k, v, 4.0, only=set(range(2 * n, 3 * n)))
            within(out[2 * n :], want[2 * n :], (ob + (want.abs() + ob) * ref.half_step(t))[2 * n :], "out")
            within(lse[2 * n :], wlse[2 * n :], lb[2 * n :], "lse")


def test_pages_from_the_library_are_ready(yl, torch_cuda):
    """The allocation's zeros are there when it returns: none are on their way that another stream's tokens could meet."""
    side = torch.cuda.Stream()
    g = ref.Geometry(63, 4, 2, 64, page=64, lens=[5], rows=[5])
    n = 1 << 17
    g.table[0, 0] = n - 1
    batch, qkv = g.device(yl), torch.full((5, 8 * 64), 3.0, device="cuda")
    ones, out = torch.ones(5, 4, 64, device="cuda"), torch.empty(5, 4, 64, device="cuda")
    torch.cuda.synchronize()
    pages = yl.KvPages.alloc(yl.DType.F32, n, 64, 2, 64)  # 4 GiB each of keys and values
    assert torch.cuda.default_stream().query()
    with torch.cuda.stream(side):
        yl.paged_append(qkv, pages, batch, 4)
        ws = torch.empty(yl.paged_attention_workspace(pages, batch, 4), dtype=torch.uint8, device="cuda")
        yl.paged_attention(out, ones, pages, batch, 4, 0.125, ws)
    torch.cuda.synchronize()
    assert (out == 3.0).all()
    pages.free()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [40, 1889, 16000, 128256])
def test_logprobs_with_few_terms_left(yl, torch_cuda, dtype, vocab):
    """Rows whose probability besides the likeliest token's lies in one to four others, 0.5 to 40 below it: the log
    probability of that token and the entropy to f32's last bits. A term is off by the exponential (4 half steps of f32,
    2^-22), the factor's product and its argument's rounding (2), a sum of four (3), log1p (2) and the sums of a thread's
    own terms next to larger ones (at most |d| e^-d 4, below 2): 13 half steps, and the last subtraction of the entropy,
    of which W / S is as large as S' at least and has 4 more, two more."""
    t = DTYPES[dtype]
    rng = np.random.default_rng(vocab)
    n = 300
    x = np.full((n, vocab), -np.inf)
    at = np.zeros(n, np.int64)
    for i in range(n):
        place = rng.permutation(vocab)[:5]
        at[i] = place[0]
        x[i, place[0]] = rng.normal() * 3 + 8
        for p in place[1 : 2 + i % 4]:
            x[i, p] = x[i, place[0]] - rng.uniform(0.5, 40)
    x = torch.from_numpy(x).to(t)
    d = x.double() - x.double().gather(1, torch.from_numpy(at)[:, None])
    e = d.exp()
    e[torch.arange(n), torch.from_numpy(at)] = 0.0
    s, w = e.sum(1), torch.where(e > 0, e * d, 0.0).sum(1)
    lp, en, ids, _ = run_logprobs(yl, x.cuda(), torch.from_numpy(at.astype(np.int32)).cuda(), 1)
    likely = s < 0.4  # (from 1/2 on S' is what S = 1 + S' has kept)
    assert int(likely.sum()) > n // 2 and np.array_equal(ids[:, 0].numpy(), at)
    within(lp[likely], -s.log1p()[likely], (13 * ref.U32 * s)[likely], "logprobs")
    within(en[likely], (s.log1p() - w / (1 + s))[likely], (19 * ref.U32 * (s - w))[likely], "entropy")
