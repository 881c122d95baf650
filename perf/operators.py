"""The key/value cache in 8 bits, as cases that can be timed one by one: rows of q, k and v rotated and appended to a paged
cache (`rope_append`), and attention over such a cache (`paged_attention`).

The cache is four tensors: k and v [pages, kv_heads, page, head_dim] in int8 or float8_e4m3fn, and their scales
[pages, kv_heads] in fp32, one for the tokens of a page and a head. Page j of sequence i is page_table[i, j]; lengths[i] is
how many tokens sequence i has in the cache, the rows of the call included; rows query_start[i] .. query_start[i + 1] of the
call are its last ones (without query_start every sequence has one row). Scales written by the append are powers of two: the
smallest with which the page's values fit the type, never smaller than what the page had when it already held tokens.

A case says: the operator; how many sequences; the most rows of a sequence (`rows`; 1 is decoding) and the most tokens of one
(`context`); whether sequences differ (`ragged`); heads, head size, page size and types. Row counts and lengths follow from
these alone, so the work of a case is known without its inputs; pages lie in the cache in an order made from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
ACTIVATIONS = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}          # the largest value of the type
LOWEST = -64                                  # exponent of the smallest scale


def _case(name, op, sequences, rows, context, heads, kv_heads, head_dim, page, cache, dtype, ragged=False):
    c = {"op": op, "sequences": sequences, "rows": rows, "context": context, "ragged": ragged, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "cache": cache, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one sequence of the Llama-2-7B-shaped decoder: what is left is the call
        _case("append_token", "append", 1, 1, 201, 32, 32, 128, 32, "int8", "fp16"),
        # 64 sequences decoded side by side, grouped heads
        _case("append_batch_64", "append", 64, 1, 4096, 32, 8, 128, 16, "fp8", "bf16", True),
        # a long prompt in one piece
        _case("append_prompt", "append", 1, 8192, 8192, 32, 8, 128, 64, "fp8", "fp16"),
        # prompts and continuations of odd lengths in one call, small heads
        _case("append_mixed_odd", "append", 13, 257, 1111, 12, 4, 64, 32, "int8", "bf16", True),
        # one token over a short context: latency
        _case("attend_token", "attend", 1, 1, 201, 32, 32, 128, 32, "int8", "fp16"),
        # 64 sequences decoded side by side, every head with keys of its own: the largest read
        _case("attend_batch_64", "attend", 64, 1, 4096, 32, 32, 128, 32, "fp8", "fp16", True),
        # one sequence with a very long context
        _case("attend_long", "attend", 1, 1, 131072, 32, 8, 128, 64, "fp8", "bf16"),
        # a few drafted tokens per sequence, checked together
        _case("attend_drafts", "attend", 16, 5, 8000, 32, 8, 128, 16, "int8", "fp16", True),
        # a prompt attending to itself
        _case("attend_prompt", "attend", 1, 4096, 4096, 32, 32, 128, 32, "fp8", "fp16"),
        # pieces of prompts behind what the cache already holds
        _case("attend_chunk", "attend", 4, 512, 16384, 32, 8, 128, 64, "int8", "bf16", True),
        # prompts and continuations of odd lengths in one call, small heads
        _case("attend_mixed_odd", "attend", 13, 777, 2001, 12, 4, 64, 16, "fp8", "fp16", True),
        # wide heads
        _case("attend_wide_heads", "attend", 5, 300, 3000, 8, 2, 256, 128, "int8", "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("append", "attend")}
    while True:
        op = rng.choice(("append", "attend", "attend"))
        kv_heads = rng.choice((1, 2, 4, 8, 32))
        heads = kv_heads * rng.choice((1, 2, 4, 8) if kv_heads < 32 else (1,))
        sequences = _log_int(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        context = max(rows, _log_int(rng, 1, 131072))
        c = _case(None, op, sequences, rows, context, heads, kv_heads, rng.choice((64, 128, 128, 256)),
                  rng.choice((16, 32, 64, 128)), rng.choice(("int8", "fp8")), rng.choice(("fp16", "bf16")), rng.random() < 0.6)
        tokens, fits = sequences * context * kv_heads * c["head_dim"], sequences * rows * (heads + 2 * kv_heads) * c["head_dim"]
        scores = sequences * heads * rows * context
        if _cost(c) <= most[op] and tokens <= 1 << 30 and fits <= 1 << 27 and (op == "append" or scores <= 1 << 30):
            return c


def _power(e):
    """2^e in fp32, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _spread(i):
    return (0.5 + 0.6180339887498949 * i) % 1.0


def _sequences(case):
    """(rows, tokens) of every sequence: the first has the most of both; where they differ, the others are spread below."""
    got = []
    for i in range(case["sequences"]):
        rows, context = case["rows"], case["context"]
        if case["ragged"] and i:
            rows = 1 + int((rows - 1) * _spread(i))
            context = max(rows, int(context * (0.05 + 0.95 * _spread(3 * i + 1))))
        got.append((rows, context))
    return got


def work(case):
    d, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    seqs = _sequences(case)
    n = sum(r for r, _ in seqs)
    if case["op"] == "append":
        longest = max(t for _, t in seqs) - min(t - r for r, t in seqs)   # positions whose table rows are read
        return {"bytes": 2 * n * (hq + 2 * hkv) * d + 2 * n * hq * d + 2 * n * hkv * d + 4 * min(n, longest) * d,
                "flops": 3 * n * (hq + hkv) * d}
    pages = sum(-(-t // case["page"]) for _, t in seqs)
    seen = sum(r * (t - r) + r * (r + 1) // 2 for r, t in seqs)
    return {"bytes": 4 * n * hq * d + 2 * sum(t for _, t in seqs) * hkv * d + 8 * pages * hkv, "flops": 4 * seen * hq * d}


def _cost(case):
    """Microseconds at 6.5 TB/s and 1.6 PFLOP/s: for the limit on drawn cases."""
    w = work(case)
    return max(w["bytes"] / 6.5e6, w["flops"] / 1.6e9)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    d, hq, hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    seqs = _sequences(case)
    counts = [-(-t // page) for _, t in seqs]
    pages, width = sum(counts), max(counts)
    # pages of the cache in any order, as a server hands them out; entries behind a sequence's last page are zero
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first = torch.tensor([sum(counts[:i]) for i in range(len(counts))], device=DEV)
    number = torch.tensor(counts, device=DEV)
    column = torch.arange(width, device=DEV)
    table = torch.where(column < number[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], 0).to(torch.int32)
    shape = (pages, hkv, page, d)

    def codes():
        # values of about unit size, the page's largest within a factor of two of the type's largest
        x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
        if case["cache"] == "int8":
            return x.mul_(26).round_().clamp_(-127, 127).to(torch.int8)
        return x.mul_(90).clamp_(-448, 448).to(torch.float8_e4m3fn)

    def scales():
        e = torch.randint(-1, 2, (pages, hkv), generator=g, device=DEV)
        return _power(e - (5 if case["cache"] == "int8" else 7))

    s = {"case": case, "k": codes(), "v": codes(), "k_scale": scales(), "v_scale": scales(), "table": table,
         "lengths": torch.tensor([t for _, t in seqs], dtype=torch.int32, device=DEV),
         "rows": max(r for r, _ in seqs), "start": None}
    n = sum(r for r, _ in seqs)
    if case["rows"] > 1:
        s["start"] = torch.tensor([sum(r for r, _ in seqs[:i]) for i in range(len(seqs) + 1)], dtype=torch.int32, device=DEV)
    dtype = ACTIVATIONS[case["dtype"]]
    if case["op"] == "append":
        x = torch.randn(n, hq + 2 * hkv, d, generator=g, device=DEV)
        x[:, :, :: d // 4] *= 4.0                                    # a few dimensions of keys are larger than the rest
        s["qkv"] = x.to(dtype).view(n, -1)
        inv = 10000.0 ** (-torch.arange(d // 2, device=DEV, dtype=torch.float64) / (d // 2))
        angle = torch.arange(width * page, device=DEV, dtype=torch.float64)[:, None] * inv
        angle = torch.cat((angle, angle), dim=-1)
        s["cos"], s["sin"] = angle.cos().half(), angle.sin().half()
    else:
        s["q"] = (2.0 * torch.randn(n, hq, d, generator=g, device=DEV)).to(dtype)
    return s


def _start(s):
    """query_start in int64, also where every sequence has one row."""
    return s["start"].long() if s["start"] is not None else torch.arange(s["lengths"].numel() + 1, device=DEV)


def _rows(s, n):
    """Sequence and position of every row."""
    start, lengths = _start(s), s["lengths"].long()
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    return seq, lengths[seq] - start[seq + 1] + row


def _to_codes(x, kind):
    """The bytes of values that have been divided by their scale, rounded to nearest even."""
    return (x.round().to(torch.int8) if kind == "int8" else x.float().to(torch.float8_e4m3fn)).view(torch.uint8)


def _append_one(s, codes, scale, x, seq, pos):
    """Rows x [n, kv_heads, head_dim], in 64 bits, into one of the two caches."""
    kind, page = s["case"]["cache"], s["case"]["page"]
    at, slot = s["table"][seq, pos // page].long(), pos % page
    # exponent of the smallest scale with which the rows on a page fit: top * 2^e >= largest
    largest = torch.zeros(scale.shape, dtype=torch.float64, device=DEV).index_reduce_(0, at, x.abs().amax(-1), "amax")
    top, top_e = math.frexp(TOP[kind])
    m, e = torch.frexp(largest)
    need = _power((e - top_e + (m > top)).clamp(min=LOWEST))
    # the first page of a sequence may hold tokens already: its scale does not shrink, and they follow it where it grows
    start, lengths = _start(s), s["lengths"].long()
    begin = lengths - (start[1:] - start[:-1])
    old_page = s["table"][torch.arange(len(lengths), device=DEV), begin // page].long()
    held = begin % page
    old = torch.where(held[:, None] > 0, scale[old_page], 0.0)
    need[old_page] = torch.maximum(need[old_page], old)
    stored = codes.view(torch.uint8)
    was = stored[old_page]
    moved = _to_codes(was.view(codes.dtype).double() * (old.double() / need[old_page].double())[:, :, None, None], kind)
    keep = (torch.arange(page, device=DEV) < held[:, None])[:, None, :, None]
    stored[old_page] = torch.where(keep, moved, was)
    touched = torch.zeros(scale.shape[0], 1, dtype=torch.bool, device=DEV).index_fill_(0, at, True)
    scale.copy_(torch.where(touched, need, scale))
    stored[at, :, slot] = _to_codes(x / scale[at].double()[..., None], kind)


def _plain_append(s):
    case = s["case"]
    d, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    x = s["qkv"].view(-1, hq + 2 * hkv, d).double()
    seq, pos = _rows(s, x.shape[0])
    cos, sin = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
    qk = x[:, : hq + hkv]
    qk = qk * cos + torch.cat((-qk[..., d // 2:], qk[..., : d // 2]), dim=-1) * sin
    _append_one(s, s["k"], s["k_scale"], qk[:, hq:], seq, pos)
    _append_one(s, s["v"], s["v_scale"], x[:, hq + hkv:], seq, pos)
    return qk[:, :hq].to(s["qkv"].dtype)


def _plain_attend(s):
    case = s["case"]
    d, hq, hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].long()
    b, width, rows, group = table.shape[0], table.shape[1], s["rows"], hq // hkv
    start = _start(s)
    n = start[1:] - start[:-1]

    def dense(codes, scale):
        x = codes.view(torch.uint8)[table].view(codes.dtype).float() * scale[table][..., None, None]                       # [b, width, kv_heads, page, d]
        return x.transpose(1, 2).reshape(b, hkv, width * page, d)

    column = torch.arange(rows, device=DEV)
    padded = q.float()[(start[:-1, None] + column).clamp(max=q.shape[0] - 1)]           # [b, rows, heads, d]
    padded = padded.view(b, rows, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * rows, d)
    score = padded @ dense(s["k"], s["k_scale"]).transpose(-1, -2) * (1.0 / math.sqrt(d))
    last = (lengths - n)[:, None] + column                                             # the last token that a row sees
    unseen = torch.arange(width * page, device=DEV) > last[..., None]                  # [b, rows, tokens]
    score = score.view(b, hkv, group, rows, -1).masked_fill_(unseen[:, None, None], float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    score = score.div_(score.sum(-1, keepdim=True)).view(b, hkv, group * rows, -1)
    out = (score @ dense(s["v"], s["v_scale"])).view(b, hkv, group, rows, d).permute(0, 3, 1, 2, 4).reshape(b, rows, hq, d)
    row = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    return out[seq, row - start[seq]].to(q.dtype)


def run(s):
    if own:
        import macko_spmv_b200 as macko_spmv

        cache = (s["k"], s["v"], s["k_scale"], s["v_scale"])
        if s["case"]["op"] == "append":
            q = macko_spmv.rope_append(s["qkv"], s["cos"], s["sin"], cache, s["table"], s["lengths"], s["start"])
        else:
            return macko_spmv.paged_attention(s["q"], cache, s["table"], s["lengths"], s["start"])
    elif s["case"]["op"] == "append":
        q = _plain_append(s)
    else:
        return _plain_attend(s)
    # the cache is returned as it is held: every code next to its scale, which is exact
    return [q, s["k"], s["v"], s["k_scale"], s["v_scale"]]


def exact(case, seed):
    s = prepare(case, seed)
    d, hq, hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    group, row, out = hq // hkv, 0, []
    scale_k, scale_v = s["k_scale"].double(), s["v_scale"].double()
    for i, (n, tokens) in enumerate(_sequences(case)):
        pages = s["table"][i, : -(-tokens // page)].long()
        if case["op"] == "append":
            x = s["qkv"][row: row + n].double().view(n, hq + 2 * hkv, 2, d // 2)
            c, z = (s[t][tokens - n: tokens, : d // 2].double()[:, None] for t in ("cos", "sin"))
            turned = torch.stack((x[:, :, 0] * c - x[:, :, 1] * z, x[:, :, 1] * c + x[:, :, 0] * z), dim=2).view(n, -1, d)
            out.append(turned[:, :hq])
            for scale, rows in ((scale_k, turned[:, hq: hq + hkv]), (scale_v, x.view(n, -1, d)[:, hq + hkv:])):
                for j in range((tokens - n) // page, (tokens - 1) // page + 1):
                    lo, hi = max(0, j * page - tokens + n), min(n, (j + 1) * page - tokens + n)
                    most = rows[lo:hi].abs().amax(dim=(0, 2))
                    near = torch.floor(torch.log2(most / TOP[case["cache"]]) - 0.5).clamp(min=LOWEST)
                    new = torch.exp2(near + sum((TOP[case["cache"]] * torch.exp2(near + k) < most).double() for k in range(3)))
                    scale[pages[j]] = torch.maximum(new, scale[pages[j]]) if lo == 0 and (tokens - n) % page else new
        else:
            q = s["q"][row: row + n].double()
            unseen = torch.arange(tokens, device=DEV) > torch.arange(tokens - n, tokens, device=DEV)[:, None]
            got = torch.empty(n, hq, d, dtype=torch.float64, device=DEV)
            for h in range(hkv):
                k, v = ((s[t].view(torch.uint8)[pages, h].view(s[t].dtype).double() * s[t + "_scale"][pages, h].double()[:, None, None]).view(-1, d)[:tokens]
                        for t in ("k", "v"))
                for a in range(h * group, (h + 1) * group):
                    p = torch.softmax((q[:, a] @ k.T / math.sqrt(d)).masked_fill_(unseen, float("-inf")), dim=-1)
                    got[:, a] = p @ v
            out.append(got)
        row += n
    out = torch.cat(out)
    return [out, None, None, scale_k, scale_v] if case["op"] == "append" else out
