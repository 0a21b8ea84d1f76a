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
def test_shared_prefix_decode(yl, torch_cuda, dtype, shape, shared):
    lens = [shared + n for n in (0, 1, 5, 16, 17, 64, 90, 200, 333)]
    g = ref.Geometry(6, *shape, page=16, lens=lens, rows=[1] * 8 + [0], shared=shared, pad_rows=1)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(9, 3, 64), (8, 2, 128)])
def test_shared_prefix_prompts(yl, torch_cuda, dtype, shape):
    """Rows behind the prefix, and rows inside it (a sequence whose chunk begins before the prefix ends)."""
    g = ref.Geometry(7, *shape, page=32, lens=[96 + 70, 96 + 1, 100, 96], rows=[70, 1, 60, 96], shared=96)
    check_attention(yl, g, DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 64])
def test_f32_output_of_16_bit_cache(yl, torch_cuda, dtype, shared):
    g = ref.Geometry(8, 8, 2, 128, page=32, lens=[64 + 30, 64 + 129, 65], rows=[1, 40, 1], shared=64)
    check_attention(yl, g, DTYPES[dtype], shared=shared, out_dtype=torch.float32)


def test_long_rows(yl, torch_cuda):
    """Long sequences, split over many blocks: one token against 40000, next to short ones."""
    for dtype in ("f32", "bf16"):
        g = ref.Geometry(9, 2, 1, 64, page=64, lens=[40000, 3, 12345], rows=[1, 1, 2])
        check_attention(yl, g, DTYPES[dtype])
    g = ref.Geometry(9, 2, 1, 64, page=64, lens=[20480 + 3, 20480 + 3000], rows=[1, 2], shared=20480)
    check_attention(yl, g, torch.float16)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts(yl, torch_cuda, dtype):
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
def test_garbage_behind_the_sequences(yl, torch_cuda, dtype, bad):
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


def test_same_bits_again_and_on_another_stream(yl, torch_cuda):
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
