"""The paged 8-bit key/value cache: `rope_append` and `paged_attention` against plain implementations in 64 bits.

Tolerances. Codes and scales of the append are exact: rotation products of 11 x 11 (fp16) or 8 x 11 (bf16) bits are added to odd, so the
one rounding to 8 bits is that of the exact value. q: one rounding, eps / 2 of its type, of a value that is exact to 2^-23.
Attention: out = sum(w v) / sum(w). The product w * scale of a token's weight and its value's scale is rounded to fp16 once, relative to the row's
largest, M: off by 2^-11 of itself, or by 2^-25 M where it is subnormal. Its products with the codes are exact, sums are fp32 (some
hundred roundings of 2^-24, and 2^-21 for the exponential), and the result is rounded once more:
|error| <= ((2^-11 + 2^-14) sum(w |v|) + 2^-25 M sum |code|) / sum(w) + eps / 2 |out|.
"""
import math

import pytest
import torch

import macko_spmv_b200 as macko_spmv

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(positions, d, device="cuda"):
    inv = 10000.0 ** (-torch.arange(d // 2, device=device, dtype=torch.float64) / (d // 2))
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    angle = torch.cat((angle, angle), -1)
    return angle.cos().half(), angle.sin().half()


def _values(codes):
    return codes.view(torch.uint8).clone().view(codes.dtype).double() if codes.dtype != torch.int8 else codes.double()


def _round_codes(x, dtype):
    """float64 values, divided by their scale, to the nearest code, ties to even."""
    if dtype == torch.int8:
        return x.round().clamp(-127, 127)
    a = x.abs()
    e = torch.frexp(a)[1].clamp(min=-5)              # values in [2^(e-1), 2^e) are 2^(e-4) apart, subnormals 2^-9
    step = torch.ldexp(torch.ones_like(a), e - 4)
    return torch.copysign(((a / step).round() * step).clamp(max=448.0), x)


def _scale_for(most, dtype):
    """Smallest power of two s >= 2^-64 with most <= top * s."""
    e = -64
    while TOP[dtype] * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


class Cache:
    """A cache with garbage in it, pages in random order, and its contents as float64 codes."""

    def __init__(self, lengths, page, kv_heads, d, dtype, seed, spare=3, strided=False):
        g = _gen(seed)
        self.page, self.hkv, self.d, self.dtype = page, kv_heads, d, dtype
        counts = [-(-n // page) for n in lengths]
        pages, width = sum(counts) + spare, max(counts + [1])
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lengths), width), -7, dtype=torch.int32, device="cuda")   # behind a sequence: no page
        at = 0
        for i, c in enumerate(counts):
            self.table[i, :c] = order[at: at + c]
            at += c
        shape = (pages, 2, kv_heads, page, d)
        x = torch.randn(shape, generator=g, device="cuda")
        codes = (x * 40).round().clamp(-127, 127).to(torch.int8) if dtype == torch.int8 else (x * 100).clamp(-448, 448).to(dtype)
        scales = torch.exp2(torch.randint(-8, -4, (pages, 2, kv_heads), generator=g, device="cuda").float())
        if strided:
            self.k, self.v, self.ks, self.vs = codes[:, 0], codes[:, 1], scales[:, 0], scales[:, 1]
        else:
            self.k, self.v, self.ks, self.vs = (t.clone(memory_format=torch.contiguous_format) for t in (
                codes.view(torch.uint8)[:, 0], codes.view(torch.uint8)[:, 1], scales[:, 0], scales[:, 1]))
            self.k, self.v = self.k.view(dtype), self.v.view(dtype)

    @property
    def tensors(self):
        return (self.k, self.v, self.ks, self.vs)

    def copy(self):
        return [t.view(torch.uint8).clone() if t.element_size() == 1 else t.clone() for t in self.tensors]


def _starts(rows):
    return torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device="cuda")


def _rotated(x, cos, sin, positions):
    """x [n, heads, d] in float64, exactly (products of 22 bits, sums of two)."""
    half = x.shape[-1] // 2
    c, s = cos[positions].double()[:, None], sin[positions].double()[:, None]
    return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * s


def _append_plain(cache, before, qkv, rows, lengths, cos, sin, hq):
    """What the four tensors of the cache have to hold afterwards (codes as float64 values), and q in float64."""
    page, hkv, d, dtype = cache.page, cache.hkv, cache.d, cache.dtype
    k, v = (_values(t.view(dtype)) for t in before[:2])
    ks, vs = before[2].double(), before[3].double()
    x = qkv.double().view(qkv.shape[0], hq + 2 * hkv, d)
    q = torch.zeros(qkv.shape[0], hq, d, dtype=torch.float64, device="cuda")
    capacity, row = cache.table.shape[1] * page, 0
    for i, (n, length) in enumerate(zip(rows, lengths)):
        by_page = {}
        for j in range(n):
            pos = length - n + j
            if 0 <= pos < capacity:
                by_page.setdefault(pos // page, []).append((row + j, pos))
        for ordinal, members in by_page.items():
            at = torch.tensor([m[0] for m in members], device="cuda")
            pos = torch.tensor([m[1] for m in members], device="cuda")
            turned = _rotated(x[at][:, : hq + hkv], cos, sin, pos)
            q[at] = turned[:, :hq]
            number = int(cache.table[i, ordinal])
            if not 0 <= number < k.shape[0]:
                continue
            slot = members[0][1] % page
            for codes, scale, new in ((k, ks, turned[:, hq:]), (v, vs, x[at][:, hq + hkv:])):
                for h in range(hkv):
                    most = float(new[:, h].abs().max())
                    old = float(scale[number, h]) if slot else 0.0
                    if not math.isfinite(float(new[:, h].abs().sum())) or math.isnan(old):
                        scale[number, h] = float("nan")
                        codes[number, h, slot: slot + len(members)] = 0
                        continue
                    now = max(_scale_for(most, dtype), old)
                    if slot and now != old:
                        codes[number, h, :slot] = _round_codes(codes[number, h, :slot] * (old / now), dtype)
                    codes[number, h, slot: slot + len(members)] = _round_codes(new[:, h] / now, dtype)
                    scale[number, h] = now
        row += n
    return k, v, ks, vs, q


def _check_append(cache, rows, lengths, hq, dtype, seed, start="given", scale_up=1.0, extra_rows=0, edit=None, tables=None):
    g = _gen(seed)
    n = sum(rows) + extra_rows
    width = (hq + 2 * cache.hkv) * cache.d
    x = torch.randn(n, hq + 2 * cache.hkv, cache.d, generator=g, device="cuda") * scale_up
    qkv = x.to(dtype).view(n, width)
    if edit is not None:
        edit(qkv)
    cos, sin = tables or _tables(cache.table.shape[1] * cache.page, cache.d)
    before = cache.copy()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = macko_spmv.rope_append(qkv, cos, sin, cache.tensors, cache.table, lens, _starts(rows) if start == "given" else None)
    k, v, ks, vs, q64 = _append_plain(cache, before, qkv, rows, lengths, cos, sin, hq)
    assert torch.equal(cache.ks.double().nan_to_num(-1.0), ks.nan_to_num(-1.0))
    assert torch.equal(cache.vs.double().nan_to_num(-1.0), vs.nan_to_num(-1.0))
    assert torch.equal(_values(cache.k), k) and torch.equal(_values(cache.v), v)
    assert q.shape == (n, hq, cache.d) and q.dtype == dtype
    far = (q.double() - q64).abs() - (torch.finfo(dtype).eps / 2 + 2.0 ** -22) * q64.abs()
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    ok = (far <= tiny) | (q64.isnan() & q.isnan()) | (q.double() == q64)
    assert bool(ok.all())
    return q


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page,hq,hkv", [(64, 16, 6, 2), (128, 32, 4, 4), (128, 64, 8, 1), (256, 128, 4, 2), (64, 128, 3, 3), (256, 16, 2, 1)])
def test_append(code, dtype, d, page, hq, hkv):
    rows = [1, 5, page, 2 * page + 3, page - 1, 1]
    lengths = [1, page + 2, page, 5 * page - 1, 3 * page + page // 2, 7 * page]
    cache = Cache(lengths, page, hkv, d, CODES[code], seed=d + page, strided=page == 32)
    _check_append(cache, rows, lengths, hq, TYPES[dtype], seed=hq)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_append_one_row_each(code):
    lengths = [1, 2, 16, 17, 31, 33, 40, 640, 0, 5]
    cache = Cache(lengths, 16, 4, 128, CODES[code], seed=3)
    _check_append(cache, [1] * len(lengths), lengths, 8, torch.float16, seed=4, start="none")


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_token_by_token_moves_a_page_to_larger_scales(code, dtype):
    """A page that fills one token at a time, tokens up to 2^12 times as large as the first: the scale grows again and again, and never shrinks."""
    cache = Cache([40], 32, 2, 64, CODES[code], seed=5)
    seen = []
    for t, size in enumerate([1e-3, 1e-3, 2e-3, 0.5, 0.1, 3.0, 1.0, 0.0, 7.0, 1e-4] + [1.0] * 25):
        _check_append(cache, [1], [t + 1], 2, TYPES[dtype], seed=100 + t, scale_up=size, start="none" if t % 2 else "given")
        if t < 32:
            seen.append(float(cache.vs[int(cache.table[0, 0]), 0]))
    assert seen == sorted(seen) and len(set(seen)) >= 4


@pytest.mark.gpu
def test_append_many_sequences():
    """More sequences than threads of a block, empty ones among them."""
    rows = [(7 * i) % 4 for i in range(700)]
    lengths = [r + (13 * i) % 50 if r else 0 for i, r in enumerate(rows)]
    cache = Cache(lengths, 16, 1, 64, torch.int8, seed=6)
    _check_append(cache, rows, lengths, 2, torch.float16, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_append_leaves_out_what_has_no_place(code):
    """Rows at negative positions, behind the table, on a page number that is none, and rows of no sequence."""
    page = 16
    lengths = [3, 40, 20, 0]
    cache = Cache([16, 32, 32, 16], page, 2, 64, CODES[code], seed=8)      # the table names two pages: 32 positions
    cache.table[2, 1] = 10 ** 6
    cache.table[2, 0] = -1
    _check_append(cache, [5, 12, 20, 2], lengths, 4, torch.float16, seed=9, extra_rows=3)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_append_of_values_that_are_not_finite(code, bad):
    cache = Cache([64, 64], 16, 2, 64, CODES[code], seed=10)

    def edit(qkv):
        qkv.view(40, 8, 64)[25, 5, 3] = bad      # a key of the second sequence, head 1
        qkv.view(40, 8, 64)[18, 6, 9] = bad      # a value of the first, head 0, on its second page

    cos, sin = _tables(64, 64)
    _check_append(cache, [20, 20], [20, 30], 4, torch.float16, seed=11, edit=edit, tables=(cos, sin))
    number = int(cache.table[0, 1])
    assert math.isnan(float(cache.vs[number, 0])) and not math.isnan(float(cache.vs[number, 1]))
    _check_append(cache, [1, 1], [21, 31], 4, torch.float16, seed=12)      # the page stays as it is, NaN
    assert math.isnan(float(cache.vs[number, 0]))
    _check_append(cache, [3, 3], [19, 19], 4, torch.float16, seed=13)      # started anew
    assert not math.isnan(float(cache.vs[number, 0]))


@pytest.mark.gpu
def test_append_extremes():
    """Zeros, the largest fp16 numbers, values at the borders of a scale and between two codes."""
    for code in (torch.int8, torch.float8_e4m3fn):
        cache = Cache([32], 32, 1, 64, code, seed=14)
        one = (torch.ones(32, 64, device="cuda").half(), torch.zeros(32, 64, device="cuda").half())

        def edit(qkv):
            x = qkv.view(12, 3, 64)
            x[:] = 0
            x[0, 1:] = torch.arange(64, device="cuda").half() - 31.5         # ties between codes at scale 1
            x[1, 1:, 0] = 127.0
            x[2, 1:, 0] = 448.0
            x[3, 1:] = torch.linspace(-448, 448, 64, device="cuda").half()
            x[4, 1, 5] = 65504.0
            x[5, 2, 5] = 127.0625

        for upto in (1, 2, 3, 4, 6, 12):
            c = Cache([32], 32, 1, 64, code, seed=14)
            _check_append(c, [upto], [upto], 1, torch.float16, seed=15, tables=one, extra_rows=12 - upto, edit=edit)


def _attend_plain(q, cache, rows, lengths, scale):
    """(out, sum(w |v|) / sum(w), M sum |code| / sum(w)) in float64, row by row of the call."""
    n, hq, d = q.shape
    out, weight, small = (torch.zeros(n, hq, d, dtype=torch.float64, device="cuda") for _ in range(3))
    group, capacity, row = hq // cache.hkv, cache.table.shape[1] * cache.page, 0
    kc, vc = _values(cache.k), _values(cache.v)
    for i, (m, length) in enumerate(zip(rows, lengths)):
        seen = max(0, min(length, capacity))
        if m and seen:
            number = cache.table[i, : -(-seen // cache.page)].long()
            there = (number >= 0) & (number < kc.shape[0])
            number = torch.where(there, number, 0)
            k = (kc[number] * cache.ks[number].double()[..., None, None]).transpose(0, 1).reshape(cache.hkv, -1, d)[:, :seen]
            codes = vc[number].transpose(0, 1).reshape(cache.hkv, -1, d)[:, :seen]
            vs = cache.vs[number].double().transpose(0, 1).repeat_interleave(cache.page, dim=1)[:, :seen]
            v = codes * vs[..., None]
            there = there.repeat_interleave(cache.page)[:seen]
            token = torch.arange(seen, device="cuda")
            pos = torch.arange(length - m, length, device="cuda")
            visible = (token <= pos[:, None]) & there
            v = torch.where(visible.any(0)[None, :, None], v, 0.0)
            for h in range(hq):
                s = (q[row: row + m, h].double() @ k[h // group].T * scale).masked_fill(~visible, float("-inf"))
                w = torch.where(visible, (s - s.amax(-1, keepdim=True)).exp(), 0.0)
                total = w.sum(-1, keepdim=True)
                total = torch.where(total == 0, 1.0, total)
                out[row: row + m, h] = w @ v[h // group] / total
                weight[row: row + m, h] = w @ v[h // group].abs() / total
                most = torch.where(visible, w * vs[h // group], 0.0).amax(-1, keepdim=True)
                small[row: row + m, h] = most * (visible.double() @ torch.where(visible.any(0)[:, None], codes[h // group].abs(), 0.0)) / total
        row += m
    return out, weight, small


def _check_attend(cache, rows, lengths, hq, dtype, seed, start="given", sharp=2.0, extra_rows=0, scale=None, q=None):
    n = sum(rows) + extra_rows
    if q is None:
        q = (torch.randn(n, hq, cache.d, generator=_gen(seed), device="cuda") * sharp).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    before = cache.copy()
    out = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, _starts(rows) if start == "given" else None, scale)
    assert out.shape == q.shape and out.dtype == dtype
    for a, b in zip(before, cache.copy()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    ref, weight, small = _attend_plain(q, cache, rows, lengths, scale if scale is not None else 1.0 / math.sqrt(cache.d))
    bound = (2.0 ** -11 + 2.0 ** -14) * weight + 2.0 ** -25 * small + torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + 2.0 ** -24
    off = (out.double() - ref).abs()
    assert bool(((off <= bound) | (ref.isnan() & out.isnan())).all()), float((off - bound).max())
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page,hq,hkv", [(64, 16, 6, 2), (128, 32, 4, 4), (128, 64, 16, 1), (256, 128, 4, 2), (64, 128, 3, 3), (256, 16, 24, 1), (128, 16, 7, 1)])
def test_attention_one_row_each(code, dtype, d, page, hq, hkv):
    lengths = [1, 2, 15, 16, 17, 127, 128, 129, 500, 0, 1033]
    cache = Cache(lengths, page, hkv, d, CODES[code], seed=d + page, strided=page == 32)
    _check_attend(cache, [1] * len(lengths), lengths, hq, TYPES[dtype], seed=hq, start="none" if d == 64 else "given")


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page,hq,hkv", [(64, 16, 6, 2), (128, 32, 4, 4), (128, 64, 8, 1), (256, 128, 4, 2), (64, 128, 3, 3), (256, 16, 5, 1), (128, 16, 7, 1)])
def test_attention_of_prompts_and_pieces(code, dtype, d, page, hq, hkv):
    rows = [1, 5, 129, 300, 64, 1, 2]
    lengths = [1, 700, 129, 300, 1000, 77, 2]
    cache = Cache(lengths, page, hkv, d, CODES[code], seed=d + page, strided=page == 32)
    _check_attend(cache, rows, lengths, hq, TYPES[dtype], seed=hq)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[2] * 9, [3, 4, 1, 2], [8], [17], [33], [130]])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (12, 1)])
def test_attention_of_a_few_rows(rows, hq, hkv):
    lengths = [r + 211 * (i + 1) for i, r in enumerate(rows)]
    cache = Cache(lengths, 32, hkv, 128, torch.int8, seed=sum(rows))
    _check_attend(cache, rows, lengths, hq, torch.float16, seed=hq)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("d,hkv,group,n", [(128, 2, 4, 1), (128, 1, 1, 1), (64, 8, 8, 1), (256, 1, 2, 1), (128, 1, 4, 40), (64, 2, 2, 200)])
def test_attention_over_a_long_context(code, d, hkv, group, n):
    cache = Cache([50001], 64, hkv, d, CODES[code], seed=21)
    _check_attend(cache, [n], [50001], hkv * group, torch.float16, seed=22)


@pytest.mark.gpu
def test_attention_of_sequences_of_very_different_length():
    lengths = [1] * 20 + [20000] + [5] * 20 + [3000, 0, 0, 700]
    cache = Cache(lengths, 16, 4, 128, torch.float8_e4m3fn, seed=23)
    _check_attend(cache, [1] * len(lengths), lengths, 8, torch.bfloat16, seed=24)
    rows = [1] * 20 + [400] + [3] * 20 + [30, 0, 2, 700]
    _check_attend(cache, rows, lengths, 8, torch.bfloat16, seed=25)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[1] * 5, [40, 3, 20, 2, 300]])
def test_attention_where_rows_see_nothing(rows):
    """Sequences that are not served, shorter than their rows, longer than their table, pages that are none, rows of no sequence."""
    lengths = [0, 2, 90, 1, 400]
    cache = Cache([16, 16, 80, 16, 320], 16, 2, 64, torch.int8, seed=26)
    cache.table[2, 1] = 1 << 30
    cache.table[4, 0] = -1
    cache.table[1, 0] = -5
    out = _check_attend(cache, rows, lengths, 4, torch.float16, seed=27, extra_rows=9)
    assert bool((out[sum(rows):] == 0).all()) and bool((out[: rows[0]] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,lengths", [([1, 1, 1], [5, 37, 100]), ([30, 1, 64], [30, 37, 100])])
def test_attention_sees_nothing_behind_the_last_token(rows, lengths):
    """NaN codes in the slots behind the last token and NaN scales on pages behind it change nothing."""
    cache = Cache(lengths, 16, 2, 128, torch.float8_e4m3fn, seed=28, spare=5)
    clean = _check_attend(cache, rows, lengths, 4, torch.float16, seed=29)
    used = set()
    for i, length in enumerate(lengths):
        for j in range(-(-length // 16)):
            number = int(cache.table[i, j])
            used.add(number)
            held = min(16, length - 16 * j)
            for t in (cache.k, cache.v):
                t.view(torch.uint8)[number, :, held:] = 0x7F
    for number in set(range(cache.k.shape[0])) - used:
        cache.ks[number] = float("nan")
        cache.vs[number] = float("inf")
        cache.v.view(torch.uint8)[number] = 0xFF
    again = macko_spmv.paged_attention((torch.randn(sum(rows), 4, 128, generator=_gen(29), device="cuda") * 2.0).half(), cache.tensors, cache.table,
                                       torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts(rows))
    assert torch.equal(clean, again)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60])
def test_attention_of_scales_that_differ_widely(n):
    """Values of pages 2^30 apart, pages of zeros with the lowest scale, keys that make the softmax pick one token."""
    lengths = [200, 200, 200]
    for code in (torch.int8, torch.float8_e4m3fn):
        cache = Cache(lengths, 16, 2, 64, code, seed=30)
        e = torch.randint(-20, 10, cache.vs.shape, generator=_gen(31), device="cuda").float()
        cache.vs.copy_(torch.exp2(e))
        number = int(cache.table[1, 2])
        cache.vs[number], cache.v.view(torch.uint8)[number] = 2.0 ** -64, 0
        _check_attend(cache, [n] * 3, lengths, 4, torch.float16, seed=32, sharp=0.2)
        cache.vs.copy_(torch.exp2(torch.randint(-9, -5, cache.vs.shape, generator=_gen(33), device="cuda").float()))
        _check_attend(cache, [n] * 3, lengths, 4, torch.bfloat16, seed=34, sharp=60.0)
        _check_attend(cache, [n] * 3, lengths, 4, torch.float16, seed=35, sharp=0.0)
        _check_attend(cache, [n] * 3, lengths, 4, torch.bfloat16, seed=35, sharp=1e-6, scale=1e5)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60])
def test_attention_to_a_page_that_is_not_finite(n):
    lengths = [100, 100]
    cache = Cache(lengths, 16, 2, 64, torch.int8, seed=36)
    q = (torch.randn(2 * n, 4, 64, generator=_gen(37), device="cuda")).half()
    lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts([n, n])
    clean = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
    cache.vs[int(cache.table[0, 1]), 1] = float("nan")
    cache.ks[int(cache.table[1, 0]), 0] = float("nan")
    out = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
    assert bool(out[:n, 2:].isnan().all()) and torch.equal(out[:n, :2], clean[:n, :2])
    assert bool(out[n:, :2].isnan().all()) and torch.equal(out[n:, 2:], clean[n:, 2:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,lengths", [([1, 1, 1], [70, 300, 9]), ([65, 3, 9], [70, 300, 9])])
def test_strided_q_and_qkv(rows, lengths):
    cache = Cache(lengths, 32, 2, 64, torch.int8, seed=38)
    n = sum(rows)
    lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts(rows)
    wide = torch.randn(n, 5, 80, generator=_gen(39), device="cuda").half()
    q = wide[:, :4, 8:72]
    assert torch.equal(macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start),
                       macko_spmv.paged_attention(q.contiguous(), cache.tensors, cache.table, lens, start))
    swapped = torch.randn(4, n, 64, generator=_gen(40), device="cuda").half().transpose(0, 1)
    assert torch.equal(macko_spmv.paged_attention(swapped, cache.tensors, cache.table, lens, start),
                       macko_spmv.paged_attention(swapped.contiguous(), cache.tensors, cache.table, lens, start))
    cos, sin = _tables(cache.table.shape[1] * 32, 64)
    qkv = torch.randn(n, 8 * 64 + 24, generator=_gen(41), device="cuda").half()[:, 16: 16 + 8 * 64]
    a = macko_spmv.rope_append(qkv, cos, sin, cache.tensors, cache.table, lens, start)
    first = cache.copy()
    b = macko_spmv.rope_append(qkv.contiguous(), cos, sin, cache.tensors, cache.table, lens, start)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(first, cache.copy()))
    wide_table = torch.full((3, cache.table.shape[1] + 5), 1 << 20, dtype=torch.int32, device="cuda")
    wide_table[:, : cache.table.shape[1]] = cache.table
    part = wide_table[:, : cache.table.shape[1]]
    assert torch.equal(macko_spmv.paged_attention(q, cache.tensors, part, lens, start), macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 20, 90])
def test_scales_of_the_softmax(d, n):
    """Negative and zero ones: the largest weight may be that of the smallest product, and all weights may be the same."""
    lengths = [n + 300, n + 1]
    cache = Cache(lengths, 32, 2, d, torch.int8, seed=d + n)
    for scale in (-0.25, 0.0, 1e-3):
        _check_attend(cache, [n, n], lengths, 4, torch.float16, seed=1, scale=scale)
        _check_attend(cache, [n, n], lengths, 4, torch.bfloat16, seed=2, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq", [(64, 300), (128, 257), (256, 130)])
@pytest.mark.parametrize("n", [1, 3])
def test_more_heads_than_a_unit_holds(d, hq, n):
    lengths = [n + 70, n]
    cache = Cache(lengths, 16, 1, d, torch.float8_e4m3fn, seed=d)
    _check_attend(cache, [n, n], lengths, hq, torch.float16, seed=3, start="none" if n == 1 else "given")
    _check_append(cache, [n, n], lengths, hq, torch.bfloat16, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_rows_of_no_sequence(d):
    cache = Cache([40], 16, 2, d, torch.int8, seed=5)
    out = _check_attend(cache, [40], [40], 4, torch.float16, seed=6, extra_rows=300)
    assert bool((out[40:] == 0).all())
    none, zero = torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.randn(500, 4, d, device="cuda").half()
    assert bool((macko_spmv.paged_attention(q, cache.tensors, cache.table[:0], none, zero) == 0).all())
    # rows in front of the first sequence's
    lens, start = torch.tensor([40], dtype=torch.int32, device="cuda"), torch.tensor([460, 500], dtype=torch.int32, device="cuda")
    late = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
    alone = macko_spmv.paged_attention(q[460:], cache.tensors, cache.table, lens, start - 460)
    assert bool((late[:460] == 0).all()) and torch.allclose(late[460:].float(), alone.float(), rtol=2e-3, atol=2e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_sizes_of_prompts(d):
    """Every number of tiles, of rows in the last unit and of pieces that a few hundred rows can have; twice, since what several warps hand one
    another must not depend on who is first."""
    for n in (41, 64, 65, 127, 128, 129, 190, 192, 255, 256, 257, 320, 385, 511, 700):
        for before in (0, 1, 63, 64, 500):
            lengths = [n + before, n]
            cache = Cache(lengths, 64, 1, d, torch.int8, seed=n)
            lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts([n, n])
            q = torch.randn(2 * n, 2, d, generator=_gen(n), device="cuda").half()
            first = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
            assert torch.equal(first, macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start))
            _check_attend(cache, [n, n], lengths, 2, torch.float16, seed=n, q=q)


@pytest.mark.gpu
def test_plain_calls_and_the_operators_agree():
    lengths = [300, 17, 64]
    a, b = (Cache(lengths, 16, 2, 64, torch.int8, seed=55) for _ in range(2))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cos, sin = _tables(a.table.shape[1] * 16, 64)
    qkv = torch.randn(3, 8 * 64, generator=_gen(56), device="cuda").half()
    versions = [t._version for t in a.tensors]
    q = macko_spmv.rope_append(qkv, cos, sin, a.tensors, a.table, lens)
    assert all(t._version > v for t, v in zip(a.tensors, versions))          # PyTorch knows that the cache was written
    r = torch.ops.macko_spmv.rope_append(qkv, cos, sin, *b.tensors, b.table, lens)
    assert torch.equal(q, r) and all(torch.equal(x, y) for x, y in zip(a.copy(), b.copy()))
    out = macko_spmv.paged_attention(q, a.tensors, a.table, lens)
    assert torch.equal(out, torch.ops.macko_spmv.paged_attention(q, *b.tensors, b.table, lens))
    assert torch.equal(out, macko_spmv.paged_attention(q, macko_spmv.KVCache(*a.tensors), a.table, lens, None, 0.125))
    assert torch.equal(out, macko_spmv.paged_attention(q, list(a.tensors), a.table, lens, scale=0.125))


@pytest.mark.gpu
def test_from_two_threads_at_once():
    import threading

    lengths = [2000, 900]
    cache = Cache(lengths, 32, 4, 128, torch.int8, seed=57)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(2, 8, 128, generator=_gen(58 + i), device="cuda").half() for i in range(2)]
    many = torch.randn(400, 8, 128, generator=_gen(60), device="cuda").half()
    start = torch.tensor([0, 300, 400], dtype=torch.int32, device="cuda")
    expected = [macko_spmv.paged_attention(q, cache.tensors, cache.table, lens) for q in qs]
    expected_many = macko_spmv.paged_attention(many, cache.tensors, cache.table, lens, start)
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                out = macko_spmv.paged_attention(qs[i], cache.tensors, cache.table, lens)
                all_rows = macko_spmv.paged_attention(many, cache.tensors, cache.table, lens, start)
                stream.synchronize()
                if not (torch.equal(out, expected[i]) and torch.equal(all_rows, expected_many)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.gpu
def test_nothing_to_do():
    cache = Cache([16], 16, 2, 64, torch.int8, seed=42)
    cos, sin = _tables(16, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    before = cache.copy()
    qkv = torch.empty(0, 8 * 64, dtype=torch.float16, device="cuda")
    q = macko_spmv.rope_append(qkv, cos, sin, cache.tensors, cache.table[:0], none)
    assert q.shape == (0, 4, 64)
    assert macko_spmv.paged_attention(q, cache.tensors, cache.table[:0], none).shape == (0, 4, 64)
    # rows, but no sequence; a sequence, but no row; a table without pages
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = torch.randn(3, 8 * 64, device="cuda").half()
    q = macko_spmv.rope_append(rows, cos, sin, cache.tensors, cache.table[:0], none, zero)
    assert bool((q == 0).all())
    assert bool((macko_spmv.paged_attention(rows[:, : 4 * 64].reshape(3, 4, 64), cache.tensors, cache.table[:0], none, zero) == 0).all())
    two = torch.zeros(2, dtype=torch.int32, device="cuda")
    macko_spmv.rope_append(rows, cos, sin, cache.tensors, cache.table, zero + 16, two)
    q = macko_spmv.rope_append(rows[:1], cos, sin, cache.tensors, cache.table[:, :0], zero + 1)
    assert bool((q == 0).all())
    assert bool((macko_spmv.paged_attention(q + 1, cache.tensors, cache.table[:, :0], zero + 1) == 0).all())
    assert all(torch.equal(x, y) for x, y in zip(before, cache.copy()))


@pytest.mark.gpu
def test_pages_beyond_32_bits():
    """A cache of more than 2^32 bytes: pages at both ends."""
    pages, page, hkv, d = (1 << 32) // (128 * 8 * 128) + 3, 128, 8, 128
    cache = Cache([130], page, hkv, d, torch.int8, seed=43)
    small = cache.copy()
    k = torch.empty((pages, hkv, page, d), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks, vs = torch.ones(pages, hkv, device="cuda"), torch.ones(pages, hkv, device="cuda")
    where = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    for big, little in zip((k, v, ks, vs), cache.tensors):
        big[where[0].long()] = little[cache.table[0].long()]
    q = torch.randn(2, 8, d, generator=_gen(44), device="cuda").half()
    for rows in ([1], [2]):
        lens, start = torch.tensor([130], dtype=torch.int32, device="cuda"), _starts(rows)
        a = macko_spmv.paged_attention(q[: rows[0]], (k, v, ks, vs), where, lens, start)
        b = macko_spmv.paged_attention(q[: rows[0]], cache.tensors, cache.table, lens, start)
        assert torch.equal(a, b)
    cos, sin = _tables(256, d)
    qkv = torch.randn(2, 24 * d, generator=_gen(45), device="cuda").half()
    macko_spmv.rope_append(qkv, cos, sin, (k, v, ks, vs), where, lens, start)
    macko_spmv.rope_append(qkv, cos, sin, cache.tensors, cache.table, lens, start)
    for big, little in zip((k, v, ks, vs), cache.tensors):
        assert torch.equal(big[where[0].long()].view(torch.uint8), little[cache.table[0].long()].view(torch.uint8))
    assert not torch.equal(small[0], cache.copy()[0])


@pytest.mark.gpu
def test_calls_repeat_exactly():
    lengths, rows = [3000, 77, 1500, 9], [400, 77, 1, 2]
    cache = Cache(lengths, 32, 2, 128, torch.float8_e4m3fn, seed=46)
    lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts(rows)
    for n, s in ((sum(rows), start), (4, None)):
        q = torch.randn(n, 8, 128, generator=_gen(47), device="cuda").half()
        first = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, s)
        for _ in range(5):
            assert torch.equal(first, macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, s))


@pytest.mark.gpu
def test_steps_together_in_a_captured_graph():
    """Append and attention as a layer runs them, captured once and replayed with other lengths and other rows; two graphs side by side."""
    page, hkv, hq, d, width = 16, 2, 4, 64, 6
    cos, sin = _tables(width * page, d)
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(3, (hq + 2 * hkv) * d, dtype=torch.float16, device="cuda")
    caches = [Cache([width * page] * 3, page, hkv, d, torch.int8, seed=48) for _ in range(2)]
    eager = Cache([width * page] * 3, page, hkv, d, torch.int8, seed=48)

    def step(cache):
        q = macko_spmv.rope_append(qkv, cos, sin, cache.tensors, cache.table, lens)
        return macko_spmv.paged_attention(q, cache.tensors, cache.table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0]), step(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for cache in caches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(cache))
        graphs.append(graph)
    other = torch.cuda.Stream()
    for t in range(40):
        lens.copy_(torch.tensor([t + 1, max(0, t - 20), 2 * t + 1], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=_gen(500 + t), device="cuda"))
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.current_stream().wait_stream(other)
        expected = step(eager)
        assert torch.equal(outs[0], expected) and torch.equal(outs[1], expected), t
    for cache in caches:
        assert all(torch.equal(x, y) for x, y in zip(cache.copy(), eager.copy()))


@pytest.mark.gpu
def test_on_another_stream():
    lengths = [900, 30]
    cache = Cache(lengths, 32, 4, 128, torch.int8, seed=49)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 128, generator=_gen(50), device="cuda").half()
    expected = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(macko_spmv.paged_attention(q, cache.tensors, cache.table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expected) for o in outs)


@pytest.mark.gpu
def test_operators_are_traceable():
    lengths = [40, 3]
    cache = Cache(lengths, 16, 2, 64, torch.int8, seed=51)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, generator=_gen(52), device="cuda").half()
    torch.library.opcheck(torch.ops.macko_spmv.paged_attention, (q, *cache.tensors, cache.table, lens), test_utils=("test_schema", "test_faketensor"))
    cos, sin = _tables(cache.table.shape[1] * 16, 64)
    qkv = torch.randn(2, 8 * 64, generator=_gen(53), device="cuda").half()
    torch.library.opcheck(torch.ops.macko_spmv.rope_append, (qkv, cos, sin, *cache.tensors, cache.table, lens), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_refusals():
    lengths = [40, 3]
    cache = Cache(lengths, 16, 2, 64, torch.int8, seed=54)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    cos, sin = _tables(cache.table.shape[1] * 16, 64)
    qkv = torch.zeros(2, 8 * 64, dtype=torch.float16, device="cuda")
    start = _starts([1, 1])

    def attend(q=q, cache=cache.tensors, table=cache.table, lens=lens, start=None):
        return macko_spmv.paged_attention(q, cache, table, lens, start)

    def append(qkv=qkv, cos=cos, sin=sin, cache=cache.tensors, table=cache.table, lens=lens, start=None):
        return macko_spmv.rope_append(qkv, cos, sin, cache, table, lens, start)

    attend(), append(), attend(start=start), append(start=start)
    k, v, ks, vs = cache.tensors
    bad_caches = [(k[:, :, :, :32], v, ks, vs), (k, v[:, :1], ks, vs), (k.float(), v.float(), ks, vs), (k, v.view(torch.float8_e4m3fn), ks, vs),
                  (k, v, ks.half(), vs), (k, v, ks[:, :1], vs), (k.cpu(), v, ks, vs), (k[:, :, :8], v[:, :, :8], ks, vs),
                  (k.transpose(2, 3), v.transpose(2, 3), ks, vs), (k[:, :, :12].contiguous(), v[:, :, :12].contiguous(), ks, vs)]
    for call in (attend, append):
        for bad in bad_caches:
            with pytest.raises(RuntimeError):
                call(cache=bad)
        for change in (dict(table=cache.table.long()), dict(lens=lens.long()), dict(lens=lens[:1]), dict(table=cache.table[:1]), dict(lens=lens.cpu()),
                       dict(table=cache.table.t()), dict(start=start[:2]), dict(start=start.long()), dict(start=start.cpu())):
            with pytest.raises(RuntimeError):
                call(**change)
    for bad in (q.float(), q[:, :3], q[:, :, :32], q[:1], q.view(2, 256), q.transpose(1, 2), torch.zeros(2, 4, 68, dtype=torch.float16, device="cuda")[:, :, 1:65]):
        with pytest.raises(RuntimeError):
            attend(q=bad)
    with pytest.raises(RuntimeError):
        append(cos=cos[:16], sin=sin[:16])
    with pytest.raises(RuntimeError):
        append(cos=cos.float(), sin=sin.float())
    for bad in (qkv[:, : 4 * 64], qkv.float(), qkv[:, :100], qkv[:1], qkv.t()):
        with pytest.raises(RuntimeError):
            append(qkv=bad)
    with pytest.raises(NotImplementedError):
        macko_spmv.paged_attention(q.cpu(), tuple(t.cpu() for t in cache.tensors), cache.table.cpu(), lens.cpu())


def test_new_cache():
    c = macko_spmv.new_cache(3, 2, 16, 64, torch.int8, device="cpu")
    assert c.k.shape == (3, 2, 16, 64) and c.v.dtype == torch.int8 and c.k_scale.shape == (3, 2) and bool((c.v_scale == 1).all())
    for bad in (dict(page_size=8), dict(head_dim=96), dict(pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            macko_spmv.new_cache(**{**dict(pages=1, kv_heads=1, device="cpu"), **bad})
    with pytest.raises(TypeError):
        macko_spmv.new_cache(1, 1, dtype=torch.float16, device="cpu")


def test_refusals_of_the_c_entries():
    """Status codes before anything is launched: no device is needed."""
    import ctypes

    from macko_spmv_b200 import cabi

    lib, at = cabi.load(), 0x10000

    def cache(**change):
        c = cabi.KVCache(k=at, v=at, k_scale=at, v_scale=at, k_page_stride=2 * 16 * 64, v_page_stride=2 * 16 * 64, k_scale_stride=2, v_scale_stride=2,
                         pages=5, kv_heads=2, page_size=16, head_dim=64, code=0)
        for name, value in change.items():
            setattr(c, name, value)
        return c

    def rows(**change):
        r = cabi.KVRows(page_table=at, lengths=at, query_start=None, table_stride=4, table_width=4, sequences=3, rows=3)
        for name, value in change.items():
            setattr(r, name, value)
        return r

    def append(c, r, row_stride=8 * 64, qkv=at, kind=0, cos=at, q=at, heads=4):
        return lib.macko_cache_rope_append(ctypes.byref(c), ctypes.byref(r), qkv, row_stride, kind, cos, at, q, heads, None)

    def attend(c, r, q_row=4 * 64, q_head=64, q=at, kind=0, out=at, heads=4):
        return lib.macko_cache_attention(ctypes.byref(c), ctypes.byref(r), q, q_row, q_head, kind, out, heads, 1.0, at, 1 << 40, None)

    bad, askew, large = cabi.ERR_INVALID_ARGUMENT, cabi.ERR_MISALIGNED, cabi.ERR_SIZE_OVERFLOW
    for call in (append, attend):
        for change, status in ((dict(k=None), bad), (dict(v_scale=None), bad), (dict(page_size=8), bad), (dict(page_size=48), bad), (dict(head_dim=96), bad),
                               (dict(code=2), bad), (dict(pages=0), bad), (dict(kv_heads=0), bad), (dict(k_page_stride=2047), bad), (dict(v_scale_stride=1), bad),
                               (dict(k=at + 8), askew), (dict(k_page_stride=2056), askew), (dict(v_scale=at + 2), askew), (dict(pages=1 << 31), large), (dict(k_page_stride=1 << 35), large)):
            assert call(cache(**change), rows()) == status, change
        for change, status in ((dict(rows=4), bad), (dict(rows=-1), bad), (dict(sequences=-1), bad), (dict(lengths=None), bad), (dict(page_table=None), bad),
                               (dict(table_stride=3), bad), (dict(lengths=at + 2), askew), (dict(query_start=at + 1), askew), (dict(table_width=1 << 27), large),
                               (dict(query_start=at, rows=1 << 25), large), (dict(sequences=1 << 21, rows=1 << 21), large)):
            assert call(cache(), rows(**change)) == status, change
        assert call(cache(), rows(), kind=2) == bad and call(cache(), rows(), heads=5) == bad and call(cache(), rows(), heads=0) == bad
        assert call(cache(), rows(), q=None) == bad and call(cache(), rows(), q=at + 8) == askew
        assert call(cache(), rows(sequences=0, rows=0, query_start=at)) == cabi.OK
    assert append(cache(), rows(), row_stride=7 * 64) == bad and append(cache(), rows(), row_stride=8 * 64 + 4) == askew
    assert append(cache(), rows(), cos=None) == bad and append(cache(), rows(), cos=at + 4) == askew
    assert attend(cache(), rows(), q_head=68) == askew and attend(cache(), rows(), out=None) == bad
    for args in ((-1, 1, 1, 4, 2, 16, 64, 0), (1, 1, 1, 3, 2, 16, 64, 0), (1, 1, 1, 4, 2, 17, 64, 0), (1, 1 << 25, 1, 4, 2, 16, 64, 0)):
        assert lib.macko_cache_attention_workspace_bytes(*args) < 0


def _model(cache_dtype=None, sequences=1, seed=31, max_len=70, **more):
    from macko_spmv_b200 import llama_decode

    cfg = dict(hidden=256, heads=4, ffn=512, vocab=1000, layers=3, eps=1e-5, rope_theta=10000.0)
    return llama_decode.LlamaDecoder(0.5, cfg=cfg, max_len=max_len, seed=seed, cache_dtype=cache_dtype, sequences=sequences, page_size=16, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("code,far", [("int8", 0.03), ("fp8", 0.1)])
def test_decoder_with_a_cache_in_8_bits(code, far):
    """Logits of the decoder with a paged cache against those with an fp16 cache. Per layer, keys and values are off by at most half a
    step: 2^-7 of a page's largest (int8, whose scale may be twice what is needed) or 2^-4 of themselves (e4m3), errors of random sign that an
    average over tokens makes smaller; the residual stream carries them on. The bounds are those steps with their root mean square over
    sqrt(3) and two for the three layers: 2 * 2^-6 and 2 * 2^-4 / sqrt(3), rounded up."""
    with torch.no_grad():
        a, b = _model(), _model(CODES[code])
        tokens = [3, 999, 17, 0, 512, 44, 8, 250, 77, 1, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15]
        for i, tok in enumerate(tokens):
            token, pos = torch.tensor([tok], device="cuda"), torch.tensor([i], device="cuda")
            la, lb = a.logits(token, pos).float(), b.logits(token, pos).float()
            assert float((la - lb).norm() / la.norm()) < far, i


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_sequences_side_by_side(code):
    """Prompts in one pass, in pieces, and mixed with single tokens: the caches are the same bits as far as the rows are, and logits agree with
    the sequence alone to the rounding of fp16 activations (2^-11 a step, some ten steps a layer)."""
    prompts = [torch.randint(0, 1000, (n,), generator=_gen(60 + n), device="cuda") for n in (5, 33, 1, 20)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        m = _model(CODES[code], sequences=4)
        whole = m.extend(torch.cat(prompts), i32([5, 33, 1, 20]), i32([0, 5, 38, 39, 59])).float()
        alone = []
        for p in prompts:
            one = _model(CODES[code])
            alone.append(one.extend(p, i32([p.numel()]), i32([0, p.numel()])).float()[0])
        alone = torch.stack(alone)
        assert float((whole - alone).norm() / alone.norm()) < 2e-2
        m = _model(CODES[code], sequences=4)
        # first 2, 30, 0 and 19 tokens, then the rest: 3, 3, 1 and 1
        first = torch.cat([prompts[0][:2], prompts[1][:30], prompts[3][:19]])
        m.extend(first, i32([2, 30, 0, 19]), i32([0, 2, 32, 32, 51]))
        rest = torch.cat([prompts[0][2:], prompts[1][30:], prompts[2], prompts[3][19:]])
        pieces = m.extend(rest, i32([5, 33, 1, 20]), i32([0, 3, 6, 7, 8])).float()
        far = 0.03 if code == "int8" else 0.1      # a page that fills in two steps may be rounded twice
        assert float((pieces - alone).norm() / alone.norm()) < far


@pytest.mark.gpu
def test_generate_batch():
    from macko_spmv_b200 import llama_decode

    prompts = [torch.randint(0, 1000, (n,), generator=_gen(70 + n), device="cuda") for n in (9, 30, 2)]
    graph, _, _ = llama_decode.generate_batch(_model(torch.int8, sequences=3), prompts, 12)
    eager, _, _ = llama_decode.generate_batch(_model(torch.int8, sequences=3), prompts, 12, use_graph=False)
    assert graph.shape == (3, 12) and torch.equal(graph, eager)
    with pytest.raises(ValueError):
        llama_decode.generate_batch(_model(torch.int8, sequences=2), prompts, 12)
    with pytest.raises(ValueError):
        llama_decode.generate_batch(_model(torch.int8, sequences=3), prompts, 60)
    single, _, _ = llama_decode.generate(_model(torch.float8_e4m3fn), prompts[0], 12)
    again, _, _ = llama_decode.generate(_model(torch.float8_e4m3fn), prompts[0], 12, use_graph=False)
    assert torch.equal(single, again)
    assert llama_decode.generate(_model(torch.int8), prompts[1], 3, batched_prefill=True)[0].shape == (3,)
    for bad in (dict(sequences=2), dict(cache_dtype=torch.int8, fused_glue=False)):
        with pytest.raises(ValueError):
            _model(**bad)
    with pytest.raises(RuntimeError):
        _model().extend(prompts[0], None)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 50])
def test_padded_batches(n):
    """Many sequences without rows, between others and at the end, and rows behind the last one's: what a batch of fixed size is padded with."""
    rows = [0] * 40 + [n] + [0] * 70 + [n, 2, 0, 1] + [0] * 200
    lengths = [(r + 20 if r else 0) for r in rows]
    cache = Cache(lengths, 16, 2, 64, torch.int8, seed=61)
    _check_append(cache, rows, lengths, 4, torch.float16, seed=62, extra_rows=77)
    out = _check_attend(cache, rows, lengths, 4, torch.float16, seed=63, extra_rows=77)
    assert bool((out[sum(rows):] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 60])
def test_short_sequences_next_to_long_ones(n, d):
    """Shares of work that end in, before and behind a short unit's only tile, with long units between."""
    rows = [n] * 25 + [1] + [n] * 12
    lengths = [n + 1 + i % 3 for i in range(10)] + [5000, n] + [n + 130 * i for i in range(13)] + [1, 2100] + [n + i for i in range(11)]
    cache = Cache(lengths, 32, 2, d, torch.float8_e4m3fn, seed=71)
    _check_attend(cache, rows, lengths, 4, torch.float16, seed=72)
