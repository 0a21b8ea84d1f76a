"""CPU: the serving entry points refuse bad arguments with status codes (no GPU
work), and the index arithmetic that bounds what their kernels touch."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
P = 1 << 20  # a stand-in for a device address: nothing below reads it


def pages(yl, **kw):
    d = dict(dtype=1, owned=0, n_pages=4, page_size=16, n_kv_heads=2, head_size=64, page_stride=16 * 128,
             token_stride=128, head_stride=64, k=P, v=P)
    d.update(kw)
    return yl.KvPagesC(**d)


def batch(yl, **kw):
    d = dict(n_seqs=2, n_rows=2, table_stride=3, shared_len=0, row_start=P, seq_len=P, page_table=P, status=None)
    d.update(kw)
    return yl.SeqBatchC(**d)


BAD_PAGES = [(dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(head_size=96), -8), (dict(page_size=4), -8),
             (dict(page_size=24), -8), (dict(page_size=512), -8), (dict(n_kv_heads=0), -1), (dict(n_pages=0), -1),
             (dict(k=None), -1), (dict(v=None), -1), (dict(k=P + 8), -1), (dict(v=P + 2), -1),
             (dict(page_stride=16 * 128 + 4), -1), (dict(token_stride=1), -1), (dict(head_stride=32), -1),
             (dict(page_stride=1 << 40), -1)]
BAD_BATCH = [(dict(n_seqs=0), -1), (dict(n_seqs=1 << 21), -1), (dict(n_rows=(1 << 24) + 1), -1),
             (dict(table_stride=0), -1), (dict(shared_len=8), -1), (dict(shared_len=64), -6),
             (dict(shared_len=0x7FFFFF10, table_stride=1 << 30), -6), (dict(row_start=None), -1),
             (dict(seq_len=None), -1), (dict(page_table=None), -1)]


def refused(yl, rc, code):
    assert rc == code, (rc, code, yl.last_error())
    assert yl.last_error()


@pytest.mark.parametrize("pages_kw,batch_kw,code", [(p, {}, c) for p, c in BAD_PAGES] + [({}, b, c) for b, c in BAD_BATCH])
def test_bad_descriptors(yl, pages_kw, batch_kw, code):
    lib, p, b = yl.raw_lib(), pages(yl, **pages_kw), batch(yl, **batch_kw)
    n = C.c_uint64()
    refused(yl, lib.yl_paged_append(P, 512, P, 1024, p, b, 4, P, 64, 0, None), code)
    refused(yl, lib.yl_paged_attention_workspace(p, b, 4, n), code)
    refused(yl, lib.yl_paged_attention(P, 256, 1, None, P, 256, p, b, 4, 0.1, P, 1 << 30, None), code)


def test_null_descriptors(yl):
    lib, n = yl.raw_lib(), C.c_uint64()
    refused(yl, lib.yl_paged_append(P, 512, P, 1024, None, batch(yl), 4, P, 64, 0, None), -1)
    refused(yl, lib.yl_paged_append(P, 512, P, 1024, pages(yl), None, 4, P, 64, 0, None), -1)
    refused(yl, lib.yl_paged_attention_workspace(pages(yl), batch(yl), 4, None), -1)
    refused(yl, lib.yl_paged_attention_workspace(None, batch(yl), 4, n), -1)
    refused(yl, lib.yl_kv_pages_alloc(1, 4, 16, 2, 64, None), -1)
    refused(yl, lib.yl_kv_pages_alloc(1, 4, 17, 2, 64, yl.KvPagesC()), -8)
    refused(yl, lib.yl_kv_pages_free(None), -1)
    refused(yl, lib.yl_model_rope(None, C.c_void_p(), C.c_uint32()), -1)
    refused(yl, lib.yl_batch_logits(None, C.c_void_p()), -1)


@pytest.mark.parametrize("args,code", [
    (dict(n_heads=0), -8), (dict(n_heads=3), -8), (dict(n_heads=34), -8), (dict(rope_mode=2), -1), (dict(qkv=None), -1),
    (dict(qkv=P + 4), -1), (dict(qkv_stride=508), -1), (dict(qkv_stride=513), -1), (dict(q_stride=255), -1),
    (dict(q_stride=260), -1), (dict(q_out=P + 2), -1), (dict(rope_len=0), -1), (dict(rope_cs=P + 8), -1)])
def test_append_refusals(yl, args, code):
    d = dict(q_out=P, q_stride=256, qkv=P, qkv_stride=512, n_heads=4, rope_cs=P, rope_len=64, rope_mode=0)
    d.update(args)
    refused(yl, yl.raw_lib().yl_paged_append(d["q_out"], d["q_stride"], d["qkv"], d["qkv_stride"], pages(yl), batch(yl),
                                             d["n_heads"], d["rope_cs"], d["rope_len"], d["rope_mode"], None), code)


@pytest.mark.parametrize("args,code", [
    (dict(out=None), -1), (dict(out=P + 8), -1), (dict(out_stride=255), -1), (dict(out_stride=257), -1),
    (dict(out_dtype=2), -8), (dict(out_dtype=7), -8), (dict(lse=P + 2), -1), (dict(q=None), -1), (dict(q=P + 4), -1),
    (dict(q_stride=128), -1), (dict(n_heads=5), -8), (dict(n_heads=64), -8), (dict(ws=None), -1), (dict(ws=P + 16), -1),
    (dict(ws_bytes=0), -1)])
def test_attention_refusals(yl, args, code):
    d = dict(out=P, out_stride=256, out_dtype=1, lse=P, q=P, q_stride=256, n_heads=4, ws=P, ws_bytes=1 << 40)
    d.update(args)
    refused(yl, yl.raw_lib().yl_paged_attention(d["out"], d["out_stride"], d["out_dtype"], d["lse"], d["q"],
                                                d["q_stride"], pages(yl), batch(yl), d["n_heads"], 0.1, d["ws"],
                                                d["ws_bytes"], None), code)


@pytest.mark.parametrize("args,code", [
    (dict(logits=None), -1), (dict(logits=P + 2), -1), (dict(dtype=5), -1), (dict(row_stride=99), -1),
    (dict(vocab=0), -1), (dict(top_k=33), -8), (dict(vocab=20, row_stride=20, top_k=21), -1), (dict(tokens=None), -1),
    (dict(logprobs=None), -1), (dict(top_ids=None), -1), (dict(top_logprobs=None), -1), (dict(entropy=P + 1), -1),
    (dict(n_rows=1 << 25), -1)])
def test_logprobs_refusals(yl, args, code):
    d = dict(logits=P, dtype=0, row_stride=100, n_rows=2, vocab=100, tokens=P, logprobs=P, entropy=P, top_k=5, top_ids=P,
             top_logprobs=P)
    d.update(args)
    refused(yl, yl.raw_lib().yl_token_logprobs(*d.values(), None), code)


def test_empty_calls(yl):
    """No rows: nothing to do, no GPU needed."""
    lib, p, b = yl.raw_lib(), pages(yl), batch(yl, n_rows=0)
    n = C.c_uint64()
    assert lib.yl_paged_append(P, 256, P, 512, p, b, 4, P, 64, 0, None) == 0
    assert lib.yl_paged_attention_workspace(p, b, 4, n) == 0
    assert lib.yl_paged_attention(P, 256, 1, None, P, 256, p, b, 4, 0.1, P, n.value, None) == 0
    assert lib.yl_token_logprobs(P, 0, 100, 0, 100, P, P, P, 5, P, P, None) == 0
    # arrays of no rows have no address
    assert lib.yl_paged_append(None, 256, None, 512, p, b, 4, P, 64, 0, None) == 0
    assert lib.yl_paged_attention(None, 256, 1, None, None, 256, p, b, 4, 0.1, P, n.value, None) == 0
    assert lib.yl_token_logprobs(None, 0, 100, 0, 100, None, None, None, 5, None, None, None) == 0


def test_paged_share_counts_for_the_workspace(yl):
    """The option decides whether a prefix gets a pass (and its parts room); by rule a short one gets none."""
    lib, p, n = yl.raw_lib(), pages(yl, n_pages=40), C.c_uint64()
    b = batch(yl, n_seqs=4, n_rows=4, shared_len=32)
    size = {}
    for share in (0, 1, -1):
        yl.config_set("paged_share", share)
        assert lib.yl_paged_attention_workspace(p, b, 4, n) == 0
        size[share] = n.value
    assert size[0] == size[-1] < size[1]
    b = batch(yl, n_seqs=64, n_rows=64, shared_len=1 << 16, table_stride=1 << 13)
    assert lib.yl_paged_attention_workspace(p, b, 4, n) == 0
    by_rule = n.value
    yl.config_set("paged_share", 0)
    assert lib.yl_paged_attention_workspace(p, b, 4, n) == 0
    yl.config_set("paged_share", -1)
    assert n.value < by_rule


HARNESS = r"""
#include <cassert>
#include <cstdio>
#include <vector>
#include "serve.h"
using namespace yl::k;
int main() {
  // page lookups of all positions around the ends of table and pool
  for (uint32_t shift = 3; shift <= 8; ++shift) {
    const uint32_t ps = 1u << shift;
    std::vector<uint32_t> table = {5, 0, 9, 10, 0xFFFFFFFFu, 3, 1, 2, 4, 11};  // two sequences of five slots
    uint32_t none = 0;
    Seqs s{2, 0, 5, 0, &none, &none, table.data(), nullptr};
    Pages p{nullptr, nullptr, 10, shift, 3, 64, 3ull * ps * 64, 3 * 64, 64};
    for (uint32_t seq = 0; seq < 2; ++seq)
      for (uint32_t pos = 0; pos < 7 * ps; ++pos) {
        const uint32_t got = page_of(s, p, seq, pos), slot = pos / ps;
        uint32_t want = NO_PAGE;
        if (slot < 5 && table[5 * seq + slot] < 10) want = table[5 * seq + slot];
        assert(got == want);
        if (got == NO_PAGE) continue;
        for (uint32_t h = 0; h < 3; ++h) {
          const uint64_t at = slot_offset(p, got, pos, h);
          assert(at == ((uint64_t)got * ps + pos % ps) * 192 + h * 64 && at + 64 <= 10ull * ps * 192);
        }
      }
    assert(page_of(s, p, 0, 0xFFFFFFFFu) == NO_PAGE);
    // past the last position nothing is looked up, however long the table says it is
    Seqs endless = s;
    endless.table_stride = 0xFFFFFFFFu;
    assert(page_of(endless, p, 0, MAX_POS) == NO_PAGE && page_of(endless, p, 0, 0xFFFFFFFFu) == NO_PAGE);
    // offsets beyond 32 bits
    Pages big{nullptr, nullptr, 10, shift, 3, 64, 1ull << 35, 3 * 64, 64};
    assert(slot_offset(big, 9, 1, 2) == (9ull << 35) + 192 + 128);
  }
  // row ranges stay within n_rows and never run backwards
  std::vector<uint32_t> rs = {0, 3, 3, 2, 900, 7};
  Seqs s{5, 10, 1, 0, rs.data(), rs.data(), rs.data(), nullptr};
  for (uint32_t i = 0; i < 5; ++i) assert(row_begin(s, i) <= 10 && row_end(s, i) <= 10 && row_end(s, i) >= row_begin(s, i));
  assert(row_end(s, 0) == 3 && row_end(s, 2) == 3 && row_end(s, 3) == 10);
  puts("ok");
}
"""


def test_index_arithmetic(tmp_path):
    src = tmp_path / "t.cpp"
    src.write_text(HARNESS)
    exe = tmp_path / "t"
    inc = ROOT / "yallma3-mini-inference_b200" / "csrc" / "kernels"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", f"-I{inc}", "-I/usr/local/cuda/include",
                    str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "ok\n"


@pytest.fixture
def mirror(yl, monkeypatch):
    """The Python mirror on CPU tensors (whose device is -1): its checks and the library's, up to a launch."""
    import torch
    api = sys.modules[yl.__name__ + ".api"]
    for name, value in dict(_torch=torch, _dtypes={torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}, _f32=torch.float32,
                            _i32=torch.int32, _u8=torch.uint8, _device=lambda: -1, _stream_of=lambda dev: 0).items():
        monkeypatch.setattr(api, name, value)
    return yl


def mirror_batch(yl, **kw):
    import torch
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    return yl.SeqBatch(ints(3), ints(2), ints(2, 3), **{**dict(n_rows=2), **kw})


def test_pages_of_expanded_tensors(mirror):
    """Heads, tokens or pages that lie on one another are refused, not taken for others behind them; an axis of one
    entry may have any stride."""
    import torch
    yl, b = mirror, mirror_batch(mirror)
    for shape, to in (((4, 16, 1, 64), (4, 16, 2, 64)), ((4, 1, 2, 64), (4, 16, 2, 64)), ((1, 16, 2, 64), (4, 16, 2, 64))):
        k = torch.zeros(*shape).expand(*to)
        with pytest.raises(yl.YlError, match="strides"):
            yl.paged_attention_workspace(yl.KvPages.of(k, k), b, 2)
    k = torch.zeros(4, 16, 2, 64).as_strided((4, 16, 2, 64), (2048, 128, 32, 1))
    with pytest.raises(yl.YlError, match="strides"):
        yl.paged_attention_workspace(yl.KvPages.of(k, k), b, 2)
    for k in (torch.zeros(4, 16, 1, 64).as_strided((4, 16, 1, 64), (1024, 64, 1, 1)), torch.zeros(1, 16, 2, 64).expand(1, 16, 2, 64),
              torch.zeros(16, 2, 64).as_strided((1, 16, 2, 64), (0, 128, 64, 1))):
        assert yl.paged_attention_workspace(yl.KvPages.of(k, k), b, 2) > 0


@pytest.mark.parametrize("name", ["row_start", "seq_len", "page_table", "status"])
def test_batch_arrays_off_their_alignment(yl, name):
    lib, p, b, n = yl.raw_lib(), pages(yl), batch(yl, **{name: P + 2}), C.c_uint64()
    refused(yl, lib.yl_paged_append(P, 256, P, 512, p, b, 4, P, 64, 0, None), -1)
    refused(yl, lib.yl_paged_attention_workspace(p, b, 4, n), -1)
    refused(yl, lib.yl_paged_attention(P, 256, 1, None, P, 256, p, b, 4, 0.1, P, 1 << 30, None), -1)


def test_counts_that_wrap_in_32_bits(mirror):
    """Counts that C would take modulo 2^32: refused before they could name rows or positions that are not there."""
    import torch
    yl, k = mirror, torch.zeros(4, 16, 2, 64)
    for kw in (dict(n_rows=-1), dict(n_rows=2 - (1 << 32)), dict(shared_len=-16), dict(shared_len=1 << 32)):
        with pytest.raises(ValueError):
            mirror_batch(yl, **kw)
    qkv, cs = torch.zeros(2, 6 * 64), torch.zeros(32, 32, 2)
    for cs_or_address, n in ((cs, -1), (cs, 16 - (1 << 32)), (P, -1), (P, 1 << 32)):
        with pytest.raises(ValueError):
            yl.paged_append(qkv, yl.KvPages.of(k, k.clone()), mirror_batch(yl), 2, rope_cs=cs_or_address, rope_len=n)
    for shape in (None, (2,), (-1, 100), (1 - (1 << 32), 100), (2, -1)):
        with pytest.raises(ValueError):
            yl.token_logprobs(P, entropy=torch.zeros(2), shape=shape)
