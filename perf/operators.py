"""Cases that measure the serving operators: appending to a paged key/value cache, attention over it (with a prefix that
all sequences share), and token log probabilities. `run` computes them in plain torch, or, with `own`, by the library."""
import importlib
import math

import numpy as np
import torch

own = False

PKG = "yallma3-mini-inference_b200"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decoded token of the smallest model (9 heads, f32 cache): latency
        dict(name="append_1_f32", op="append", type="f32", heads=9, kv_heads=3, head_size=64, page=16, seqs=1,
             own_lo=300, own_hi=300, rows_lo=1, rows_hi=1, half=False),
        # a decode step of 64 sessions on the 8B shape
        dict(name="append_64_bf16", op="append", type="bf16", heads=32, kv_heads=8, head_size=128, page=64, seqs=64,
             own_lo=1, own_hi=500, rows_lo=1, rows_hi=1, half=True),
        # prompts of odd lengths prefilled together
        dict(name="append_prompts_f16", op="append", type="f16", heads=32, kv_heads=8, head_size=128, page=32, seqs=7,
             own_lo=900, own_hi=1500, rows_lo=700, rows_hi=1400, half=True),
        # one session, short context, f32 cache: latency
        dict(name="attend_1_f32", op="attend", type="f32", heads=9, kv_heads=3, head_size=64, page=16, seqs=1,
             shared=0, own_lo=301, own_hi=301, rows_lo=1, rows_hi=1),
        # decode of 16 sessions of uneven lengths that share nothing
        dict(name="attend_16_ragged_bf16", op="attend", type="bf16", heads=32, kv_heads=8, head_size=128, page=64,
             seqs=16, shared=0, own_lo=17, own_hi=8000, rows_lo=1, rows_hi=1),
        # decode of 64 sessions behind one long document
        dict(name="attend_64_shared_bf16", op="attend", type="bf16", heads=32, kv_heads=8, head_size=128, page=64,
             seqs=64, shared=32768, own_lo=1, own_hi=1000, rows_lo=1, rows_hi=1),
        # decode of 12 sessions behind a system prompt, f32 cache, 1B shape
        dict(name="attend_12_shared_f32", op="attend", type="f32", heads=32, kv_heads=8, head_size=64, page=32,
             seqs=12, shared=4096, own_lo=5, own_hi=900, rows_lo=1, rows_hi=1),
        # prompts of four sessions prefilled behind a shared system prompt
        dict(name="attend_prompts_f16", op="attend", type="f16", heads=32, kv_heads=8, head_size=128, page=64, seqs=4,
             shared=2048, own_lo=1100, own_hi=2100, rows_lo=1000, rows_hi=2000),
        # one long prompt, no sharing
        dict(name="attend_prompt_bf16", op="attend", type="bf16", heads=32, kv_heads=8, head_size=128, page=64, seqs=1,
             shared=0, own_lo=8191, own_hi=8191, rows_lo=8191, rows_hi=8191),
        # the sampled token of one session
        dict(name="logprobs_1_f32", op="logprobs", type="f32", rows=1, vocab=49152, top=5, masked=0.0),
        # a decode step of 64 sessions with alternatives
        dict(name="logprobs_64_f32", op="logprobs", type="f32", rows=64, vocab=128256, top=20, masked=0.1),
        # scoring of a whole prompt
        dict(name="logprobs_prompt_f32", op="logprobs", type="f32", rows=1999, vocab=128256, top=1, masked=0.0),
    ]


def _between(rng, lo, hi):
    """Log-uniform whole number."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([_between(rng, 1000, 200000), 49152, 128256])
        rows = _between(rng, 1, max(1, min(2048, 250_000_000 // vocab)))
        return dict(op=op, type=rng.choice(["f32", "f32", "f16", "bf16"]), rows=rows, vocab=vocab,
                    top=rng.choice([0, 1, 5, 20, 32]), masked=rng.choice([0.0, 0.1, 0.9]))
    heads, kv_heads, head_size = rng.choice([(9, 3, 64), (32, 8, 64), (32, 8, 128), (14, 2, 64), (8, 8, 128), (8, 1, 128)])
    c = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), heads=heads, kv_heads=kv_heads, head_size=head_size,
             page=rng.choice([8, 16, 32, 64, 128, 256]))
    kind = rng.choice(["decode", "decode", "prompt"])
    if kind == "decode":
        c.update(seqs=_between(rng, 1, 64), rows_lo=1, rows_hi=1)
        hi = _between(rng, 2, 8000 if c["seqs"] <= 16 else 1000)
    else:
        c.update(seqs=_between(rng, 1, 7))
        hi = _between(rng, 2, 2000)
        c.update(rows_lo=_between(rng, 1, hi), rows_hi=hi)
    c.update(own_lo=_between(rng, 1, hi), own_hi=hi)
    if op == "append":
        c["half"] = rng.choice([True, False])
    else:
        c["shared"] = rng.choice([0, _between(rng, 1, 16384 if kind == "decode" else 2048)]) // c["page"] * c["page"]
    return c


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], uneven, the same for every seed."""
    return [lo + int((hi - lo + 1) * ((0.5 + 0.6180339887 * i) % 1.0)) for i in range(n)]


def _lengths(case):
    """Per sequence: tokens after the shared prefix, and how many of them are new rows."""
    tokens = _spread(case["own_lo"], case["own_hi"], case["seqs"])
    return tokens, [min(t, r) for t, r in zip(tokens, _spread(case["rows_lo"], case["rows_hi"], case["seqs"]))]


def _package():
    return importlib.import_module(PKG)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = TYPES[case["type"]]
    if case["op"] == "logprobs":
        n, vocab, k = case["rows"], case["vocab"], case["top"]
        x = randn(n, vocab).mul_(2.5)
        # a few likely tokens a row, some rows nearly certain, as a model's logits have them
        likely = torch.randint(vocab, (n, 8), generator=g, device="cuda")
        x.scatter_add_(1, likely, 6 + 4 * randn(n, 8).abs())
        if case["masked"]:
            x.masked_fill_(torch.rand(n, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
        f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        return dict(op="logprobs", k=k, logits=x.to(t), tokens=likely[:, 0].int().contiguous(), logprobs=f(n),
                    entropy=f(n), top_ids=torch.empty(n, k, dtype=torch.int32, device="cuda"), top_logprobs=f(n, k))
    heads, kv_heads, hd, page = case["heads"], case["kv_heads"], case["head_size"], case["page"]
    shared = case.get("shared", 0)
    tokens, rows = _lengths(case)
    n_seqs, n_rows = len(tokens), sum(rows)
    first = shared // page  # page slots of the prefix
    need = [-(-x // page) for x in tokens]
    n_pages = first + sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    at = np.concatenate([[0], np.cumsum(need)])
    slots = np.full((n_seqs, first + max(need)), -1, np.int64)
    slots[:, :first] = np.arange(first)
    for i in range(n_seqs):
        slots[i, first : first + need[i]] = first + np.arange(at[i], at[i + 1])
    slots = torch.from_numpy(slots).cuda()
    table = torch.where(slots >= 0, order[slots.clamp(min=0)], -1).int().contiguous()
    dev = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    s = dict(op=case["op"], heads=heads, kv_heads=kv_heads, hd=hd, page=page, shared=shared, table=table,
             seq_len=dev([shared + x for x in tokens]), row_start=dev([0] + list(np.cumsum(rows))), n_rows=n_rows,
             longest=max(rows), k=randn(n_pages, page, kv_heads, hd).to(t), v=randn(n_pages, page, kv_heads, hd).to(t))
    if case["op"] == "append":
        angle = torch.arange(max(tokens), device="cuda").double()[:, None] * (
            500000.0 ** (-torch.arange(hd // 2, device="cuda").double() / (hd // 2)))
        s.update(half=case["half"], qkv=randn(n_rows, (heads + 2 * kv_heads) * hd),
                 cs=torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(),
                 q=torch.empty(n_rows, heads, hd, dtype=t, device="cuda"))
    else:
        s.update(q=(2 * randn(n_rows, heads, hd)).to(t), out=torch.empty(n_rows, heads, hd, dtype=t, device="cuda"),
                 lse=torch.empty(n_rows, heads, device="cuda"), scale=hd**-0.5)
    if own:  # the handles that a server keeps beside its cache
        yl = _package()
        s["pages"] = yl.KvPages.of(s["k"], s["v"])
        s["batch"] = yl.SeqBatch(s["row_start"], s["seq_len"], table, n_rows, shared_len=shared)
        if case["op"] == "attend":
            s["workspace"] = torch.empty(yl.paged_attention_workspace(s["pages"], s["batch"], heads), dtype=torch.uint8,
                                         device="cuda")
    return s


def _own(s):
    yl = _package()
    if s["op"] == "logprobs":
        yl.token_logprobs(s["logits"], s["tokens"], s["logprobs"], entropy=s["entropy"], top_ids=s["top_ids"],
                          top_logprobs=s["top_logprobs"])
        return {n: s[n] for n in ("logprobs", "entropy", "top_ids", "top_logprobs")}
    if s["op"] == "append":
        mode = yl.ROPE_LLAMA3 if s["half"] else yl.ROPE_GGUF
        yl.paged_append(s["qkv"], s["pages"], s["batch"], s["heads"], rope_cs=s["cs"], rope_mode=mode, q_out=s["q"])
        return {n: s[n] for n in ("q", "k", "v")}
    yl.paged_attention(s["out"], s["q"], s["pages"], s["batch"], s["heads"], s["scale"], s["workspace"], lse=s["lse"])
    return {n: s[n] for n in ("out", "lse")}


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[s["op"]](s)


def _rows(s):
    """Sequence, number within it and position of each row."""
    row = torch.arange(s["n_rows"], device="cuda")
    start = s["row_start"].long()
    seq = torch.searchsorted(start, row, right=True) - 1
    within = row - start[seq]
    return seq, within, s["seq_len"].long()[seq] - (start[seq + 1] - start[seq]) + within


def _append(s):
    heads, kv, hd = s["heads"], s["kv_heads"], s["hd"]
    seq, _, pos = _rows(s)
    x = s["qkv"].view(s["n_rows"], heads + 2 * kv, hd)
    qk = x[:, : heads + kv]
    c, sn = (s["cs"][pos][:, None, :, i] for i in (0, 1))
    if s["half"]:
        a, b = qk[..., : hd // 2], qk[..., hd // 2 :]
        qk = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    else:
        a, b = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    page, at = s["table"][seq, pos // s["page"]].long(), pos % s["page"]
    s["k"][page, at] = qk[:, heads:].to(s["k"].dtype)
    s["v"][page, at] = x[:, heads + kv :].to(s["v"].dtype)
    return {"q": qk[:, :heads].to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def _attend(s):
    kv, hd, first = s["kv_heads"], s["hd"], s["shared"] // s["page"]
    group = s["heads"] // kv
    seq, within, _ = _rows(s)
    start, length = s["row_start"].long(), s["seq_len"].long()
    n = length.numel()
    step = torch.arange(s["longest"], device="cuda")
    row = (start[:n, None] + step).clamp(max=s["n_rows"] - 1)
    q = s["q"].float().view(-1, kv, group, hd)[row] * s["scale"]  # [n, rows, kv, group, hd]
    gather = lambda pool, slots: pool[slots.clamp(min=0).long()].float().flatten(-4, -3)  # noqa: E731
    mine, all_ = s["table"][:, first:], s["table"][0, :first]
    x = torch.einsum("nrhgd,nlhd->nhgrl", q, gather(s["k"], mine))
    at = s["shared"] + torch.arange(x.shape[-1], device="cuda")
    pos = length[:, None] - (start[1:] - start[:n])[:, None] + step  # [n, rows]
    x.masked_fill_((at > pos[:, :, None])[:, None, None], -math.inf)
    if first:
        x = torch.cat([torch.einsum("nrhgd,lhd->nhgrl", q, gather(s["k"], all_)), x], -1)
    top = x.amax(-1, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    p, own_p = x[..., : s["shared"]], x[..., s["shared"] :]
    out = torch.einsum("nhgrl,nlhd->nrhgd", own_p, gather(s["v"], mine))
    if first:
        out += torch.einsum("nhgrl,lhd->nrhgd", p, gather(s["v"], all_))
    out = out / total.permute(0, 3, 1, 2, 4)
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2)
    return {"out": out[seq, within].reshape(-1, s["heads"], hd).to(s["q"].dtype),
            "lse": lse[seq, within].reshape(-1, s["heads"])}


def _logprobs(s):
    x, k = s["logits"].float(), s["k"]
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = d.exp()
    total = e.sum(-1)
    log_total = total.log()
    weighted = torch.where(e > 0, e * d, 0.0).sum(-1)
    at = lambda idx: d.gather(1, idx.long()) - log_total[:, None]  # noqa: E731
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k].int() if k else s["top_ids"]
    return {"logprobs": at(s["tokens"][:, None])[:, 0], "entropy": log_total - weighted / total, "top_ids": ids,
            "top_logprobs": at(ids) if k else s["top_logprobs"]}


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    heads, kv, hd, shared = case["heads"], case["kv_heads"], case["head_size"], case.get("shared", 0)
    tokens, rows = _lengths(case)
    n = sum(rows)
    if case["op"] == "append":
        positions = max(tokens) - min(t - r for t, r in zip(tokens, rows))
        return {"bytes": n * (heads + 2 * kv) * hd * (4 + size) + min(n, positions) * hd * 4,
                "flops": 3 * n * (heads + kv) * hd}
    seen = sum(r * (shared + t) - r * (r - 1) // 2 for t, r in zip(tokens, rows))
    return {"bytes": 2 * (shared + sum(tokens)) * kv * hd * size + 2 * n * heads * hd * size + n * heads * 4,
            "flops": 4 * seen * heads * hd}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        lp = x - lse
        del x
        best = torch.topk(lp, s["k"], -1)[0] if s["k"] else s["top_logprobs"].double()
        entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1)
        return {"logprobs": lp[torch.arange(len(lp), device="cuda"), s["tokens"].long()], "entropy": entropy,
                "top_ids": None, "top_logprobs": best if s["k"] else None}
    tokens, rows = _lengths(case)
    hd, page, heads, kv = s["hd"], s["page"], s["heads"], s["kv_heads"]
    outs = []
    r0 = 0
    for i, (t, r) in enumerate(zip(tokens, rows)):
        length = s["shared"] + t
        where = torch.arange(length, device="cuda")
        slot = s["table"][i].long()[where // page] * page + where % page
        if case["op"] == "append":
            new = where[length - r :]
            z = s["qkv"][r0 : r0 + r].double().view(r, heads + 2 * kv, hd)
            cs = s["cs"].double()[new]
            turn = torch.complex(cs[..., 0], cs[..., 1])[:, None]
            pairs = z[:, : heads + kv]
            pairs = pairs.view(r, -1, 2, hd // 2).transpose(2, 3) if s["half"] else pairs.view(r, -1, hd // 2, 2)
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            turned = (turned.transpose(2, 3) if s["half"] else turned).reshape(r, heads + kv, hd)
            outs.append((slot[length - r :], turned, z[:, heads + kv :]))
        else:
            q = s["q"][r0 : r0 + r].double()
            k, v = (s[n].view(-1, kv, hd)[slot].double() for n in ("k", "v"))
            hidden = where[None, :] > where[length - r :, None]
            out, lse = torch.empty(r, heads, hd, dtype=torch.float64, device="cuda"), torch.empty(
                r, heads, dtype=torch.float64, device="cuda")
            for h in range(heads):
                x = (q[:, h] @ k[:, h * kv // heads].T * s["scale"]).masked_fill_(hidden, -math.inf)
                lse[:, h] = torch.logsumexp(x, -1)
                out[:, h] = torch.softmax(x, -1) @ v[:, h * kv // heads]
            outs.append((out, lse))
        r0 += r
    if case["op"] == "attend":
        return {"out": torch.cat([o[0] for o in outs]), "lse": torch.cat([o[1] for o in outs])}
    k, v = s["k"].double(), s["v"].double()
    for slot, turned, value in outs:
        k.view(-1, kv, hd)[slot] = turned[:, heads:]
        v.view(-1, kv, hd)[slot] = value
    return {"q": torch.cat([o[1][:, :heads] for o in outs]), "k": k, "v": v}
