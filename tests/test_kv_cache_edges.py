"""The paged 8-bit cache at its edges: long tails of small weights and scores far from zero.

Tolerances of the attention, as in test_kv_cache.py but for the weights' fp16: the largest product of a weight with its value's scale, M, is 2^15 in fp16
in the kernel for a few rows and 2^7 to 2^15 in the one for many, so what is subnormal there is off by 2^-40 M or 2^-32 M:
|error| <= ((2^-11 + sums) sum(w |v|) + lost M sum |code|) / sum(w) + eps / 2 |out|,  lost = 2^-40 or 2^-32.

`sums` is 2^-14 where a few hundred roundings are added up. Where all values have one sign and one weight it grows with the tokens: the tensor core
adds 16 tokens at a time and cuts what falls off the fp32 sum, less than 2^-23 of it; after the k-th of n such steps the sum is k / n of the last, so
together less than n / 2 * 2^-23. The softmax sum is rounded as often, by 2^-24: n / 2 * 2^-24. With 2^-20 for the exponential and the division:
sums = 1.5 * 2^-23 * (tokens / 16) / 2 + 2^-20, which is 2^-12.5 for 30000 tokens.
"""
import math

import pytest
import torch

import macko_spmv_b200 as macko_spmv
from test_kv_cache import CODES, TYPES, Cache, _attend_plain, _check_append, _check_attend, _gen, _model, _starts

FEW, MANY = 2.0 ** -40, 2.0 ** -32


def _check(cache, rows, lengths, q, lost, scale=None, times=1, sums=2.0 ** -14):
    """`times`: the same sequences so many times over the same pages, so that there are units for all CTAs and none has to be cut."""
    lens = torch.tensor(lengths * times, dtype=torch.int32, device="cuda")
    table = cache.table.repeat(times, 1)
    out = macko_spmv.paged_attention(q.repeat(times, 1, 1), cache.tensors, table, lens, _starts(rows * times), scale)
    ref, weight, small = _attend_plain(q, cache, rows, lengths, scale if scale is not None else 1.0 / math.sqrt(cache.d))
    bound = (2.0 ** -11 + sums) * weight + lost * small + torch.finfo(q.dtype).eps / 2 * ref.abs() * 1.01 + 2.0 ** -24
    off = (out.double().view(times, *ref.shape) - ref).abs()
    assert bool(((off <= bound) | (ref.isnan() & out.view(off.shape).isnan())).all()), float((off / bound).nan_to_num(1e30).max())


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,n", [(64, 1), (128, 1), (256, 1), (128, 5), (64, 40), (128, 40), (256, 40)])
def test_one_token_with_most_of_the_weight(code, dtype, d, n):
    """One token takes 0.5 to 0.99 of the weight and has no value; tens of thousands share the rest, all the same score and values of one sign,
    so that what is lost of a weight is lost of the result."""
    tokens = 30000
    cache = Cache([tokens], 64, 4, d, CODES[code], seed=d + n)
    cache.k.view(torch.uint8)[:] = 0
    cache.v.view(torch.uint8)[:] &= 0x7D                                   # no signs, and no code that is none
    cache.ks.fill_(1.0)
    cache.vs.fill_(2.0 ** -6)
    sink = int(cache.table[0, 0])
    cache.k[sink, :, 0, 0] = 8.0
    cache.v.view(torch.uint8)[sink, :, 0] = 0
    share = torch.linspace(0.5, 0.99, 8 * n, device="cuda", dtype=torch.float64)
    nats = torch.log(share / (1 - share) * tokens)
    q = torch.zeros(n, 8, d, device="cuda", dtype=torch.float64)
    q[:, :, 0] = (nats / 8 * math.sqrt(d)).view(n, 8)
    _check(cache, [n], [tokens], q.to(TYPES[dtype]), FEW if n <= 5 else MANY, times=111, sums=1.5 * 2.0 ** -23 * tokens / 32 + 2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 60])
def test_scores_far_from_zero(code, dtype, d, n):
    """Scores of up to 2^50, where fp32 has no fractions left: the tokens that share the largest one share the result, in rows
    of ordinary scores next to them as well."""
    rows, lengths = [n, n, n], [500, 130 + n, n]
    cache = Cache(lengths, 32, 2, d, CODES[code], seed=d)
    cache.vs.fill_(2.0 ** -7)
    g = _gen(n + d)
    for codes in ([-80.0, 0.0, 80.0], [32.0, 64.0, 96.0]):
        pick = torch.randint(0, 3, cache.k.shape[:3], generator=g, device="cuda")
        cache.k.view(torch.uint8)[:] = 0
        cache.k[..., 0] = torch.tensor(codes, device="cuda")[pick].to(cache.dtype)
        for scale_k in (1.0, 2.0 ** 10, 2.0 ** 30):
            cache.ks.fill_(scale_k)
            e = torch.randint(-14, 15, (3 * n, 4), generator=g, device="cuda")
            sign = torch.randint(0, 2, e.shape, generator=g, device="cuda") * 2 - 1
            q = torch.zeros(3 * n, 4, d, device="cuda")
            q[..., 0] = sign * torch.exp2(e.float()) * 1.5
            _check(cache, rows, lengths, q.to(TYPES[dtype]), FEW if n == 1 else MANY)


def test_limit_of_waits():
    from macko_spmv_b200 import cabi

    lib = cabi.load()
    for bad in (-1, 2 * 10 ** 9 + 1, 1 << 40):
        assert lib.macko_cache_attention_wait_limit(bad) == cabi.ERR_INVALID_ARGUMENT
    for good in (0, 10 ** 6, 2 * 10 ** 9):
        assert lib.macko_cache_attention_wait_limit(good) == cabi.OK


def test_softmax_scales_that_are_not_finite_are_refused():
    """(Many rows of a NaN scale gave the mean of the values, a few rows NaN.) No device is needed."""
    import ctypes

    from macko_spmv_b200 import cabi

    lib, at = cabi.load(), 0x10000
    cache = cabi.KVCache(k=at, v=at, k_scale=at, v_scale=at, k_page_stride=2 * 16 * 64, v_page_stride=2 * 16 * 64, k_scale_stride=2, v_scale_stride=2,
                         pages=5, kv_heads=2, page_size=16, head_dim=64, code=0)
    for rows in (3, 0):
        batch = cabi.KVRows(page_table=at, lengths=at, query_start=at, table_stride=4, table_width=4, sequences=3, rows=rows)
        for scale in (math.nan, math.inf, -math.inf, 3e38):
            assert lib.macko_cache_attention(ctypes.byref(cache), ctypes.byref(batch), at, 4 * 64, 64, 0, at, 4, scale, at, 1 << 40, None) == cabi.ERR_INVALID_ARGUMENT


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_waits_that_run_out_end_the_call(d):
    """With limits of nothing, some and tens of microseconds every wait of the many-rows kernel ends, wherever the CTA is then, and the next call is
    as if nothing had been."""
    from macko_spmv_b200 import cabi

    lib = cabi.load()
    lengths, rows = [3000, 500, 64, 7], [700, 500, 64, 7]
    cache = Cache(lengths, 32, 2, d, torch.int8, seed=d)
    lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts(rows)
    q = torch.randn(sum(rows), 8, d, generator=_gen(d), device="cuda").half()
    good = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
    torch.cuda.synchronize()
    try:
        for limit in (0, 1, 300, 1000, 3000, 10000, 30000):
            assert lib.macko_cache_attention_wait_limit(limit) == cabi.OK
            for _ in range(3):
                macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
            torch.cuda.synchronize()
    finally:
        assert lib.macko_cache_attention_wait_limit(2 * 10 ** 9) == cabi.OK
    assert torch.equal(macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start), good)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths", [([700, 500, 64, 7], [3000, 500, 64, 7]), ([100] * 40, [100 + 37 * i for i in range(40)]), ([300], [20000])])
def test_rows_lost_with_a_wait_are_nan(rows, lengths, d):
    """Every row of a call whose waits run out is right or NaN in all of a head, whatever was in its place before."""
    from macko_spmv_b200 import cabi

    lib = cabi.load()
    cache = Cache(lengths, 32, 2, d, torch.int8, seed=d)
    lens, start = torch.tensor(lengths, dtype=torch.int32, device="cuda"), _starts(rows)
    q = torch.randn(sum(rows), 8, d, generator=_gen(d), device="cuda").bfloat16()
    good = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
    try:
        for limit, least in ((0, 0.9), (1, 0.9), (300, 0.0), (2000, 0.0), (8000, 0.0), (30000, 0.0)):
            assert lib.macko_cache_attention_wait_limit(limit) == cabi.OK
            for _ in range(3):
                filled = torch.full_like(q, 7.0)                       # memory that the next result is likely to get
                del filled
                out = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start)
                lost = out.isnan().all(-1)
                assert bool((lost[..., None] | (out == good)).all())
                assert float(lost.float().mean()) >= least, limit
    finally:
        assert lib.macko_cache_attention_wait_limit(2 * 10 ** 9) == cabi.OK
    assert torch.equal(macko_spmv.paged_attention(q, cache.tensors, cache.table, lens, start), good)


@pytest.mark.gpu
def test_logits_of_sequences_without_rows():
    """A padded call gives every sequence its own logits, or NaN; rows that query_start names beyond the call's are no rows. The products round
    fp16 activations in another order for another number of sequences: 2^-11 a step, some ten steps in each of three layers, 2e-2 in all."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    prompts = [torch.randint(0, 1000, (n,), generator=_gen(80 + n), device="cuda") for n in (5, 9)]
    with torch.no_grad():
        model = _model(torch.int8, sequences=4)
        logits = model.extend(torch.cat(prompts), i32(0, 5, 0, 9), i32(0, 0, 5, 5, 14))
        alone = _model(torch.int8, sequences=4)
        both = alone.extend(torch.cat(prompts), i32(5, 9), i32(0, 5, 14), alone.page_table[[1, 3]])
        assert bool(logits[[0, 2]].isnan().all())
        assert float((logits[[1, 3]] - both).float().norm() / both.float().norm()) < 2e-2
        token = torch.tensor([1, 2, 3, 4], device="cuda")
        step = model.extend(token, i32(0, 6, 0, 10))
        assert step[[0, 2]].isnan().all() and not step[[1, 3]].isnan().any()
        assert bool(model.extend(token[:0], i32(0, 6, 0, 10), i32(0, 0, 0, 0, 0)).isnan().all())
        far = model.extend(token, i32(4, 0, 0, 0), i32(0, 4, 9, 9, 9))
        assert bool(far[1:].isnan().all()) and not far[0].isnan().any()
        for tokens in (token[:0], torch.zeros(71, dtype=torch.int64, device="cuda")):
            with pytest.raises(ValueError):
                model.prefill(tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("n", [1, 60])
def test_the_largest_scales_of_values(d, n):
    """Scales of a user's own up to 2^127, with codes that keep the values inside bfloat16."""
    lengths = [n + 70, n]
    cache = Cache(lengths, 16, 2, d, torch.int8, seed=d)
    cache.v.clamp_(-1, 1)
    cache.vs.copy_(torch.exp2(torch.randint(122, 128, cache.vs.shape, generator=_gen(d), device="cuda").float()))
    _check(cache, [n, n], lengths, (torch.randn(2 * n, 4, d, generator=_gen(n), device="cuda")).bfloat16(), FEW if n == 1 else MANY)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page,hq,hkv", [(64, 16, 6, 2), (128, 32, 4, 4), (128, 64, 16, 1), (256, 128, 4, 2), (64, 128, 3, 3), (256, 16, 24, 1), (128, 16, 7, 1), (256, 64, 9, 3)])
@pytest.mark.parametrize("longest", [33, 500, 1000, 2300])
def test_one_row_each_without_query_start(code, dtype, d, page, hq, hkv, longest):
    """Decoding as it is called most: tables of up to 1024 tokens, where every unit has a CTA of its own, and longer ones. Empty sequences, ones that are
    longer than their table, and pages that are none."""
    lengths = [1, longest, 0, 2, longest // 2 + 1, longest + 5000, 16, 17, longest - 1, 0]
    cache = Cache([min(n, longest) for n in lengths], page, hkv, d, CODES[code], seed=d + page, strided=page == 32)
    cache.table[4, 0] = -3
    cache.table[8, cache.table.shape[1] // 2] = 1 << 30
    for start in ("none", "given"):
        _check_attend(cache, [1] * len(lengths), lengths, hq, TYPES[dtype], seed=hq, start=start)


@pytest.mark.gpu
@pytest.mark.parametrize("longest", [100, 3000])
def test_one_row_each_on_pages_that_are_not_finite(longest):
    lengths = [longest, 100, 90]
    cache = Cache(lengths, 16, 2, 64, torch.int8, seed=36)
    q = torch.randn(3, 4, 64, generator=_gen(37), device="cuda").half()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    clean = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens)
    cache.vs[int(cache.table[0, 1]), 1] = float("nan")
    cache.ks[int(cache.table[1, 0]), 0] = float("nan")
    out = macko_spmv.paged_attention(q, cache.tensors, cache.table, lens)
    assert bool(out[0, 2:].isnan().all()) and torch.equal(out[0, :2], clean[0, :2])
    assert bool(out[1, :2].isnan().all()) and torch.equal(out[1, 2:], clean[1, 2:])
    assert torch.equal(out[2], clean[2])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_padded_batches_of_many_rows(d):
    """Long runs of sequences without rows in front of, between and behind prompts, through the kernel for many rows (20 heads a cache head: 38 rows
    a sequence on average)."""
    rows = [0] * 40 + [300] + [0] * 70 + [300, 2, 0, 1] + [0] * 200
    lengths = [(r + 20 if r else 0) for r in rows]
    cache = Cache(lengths, 16, 2, d, torch.int8, seed=61)
    out = _check_attend(cache, rows, lengths, 40, torch.float16, seed=63, extra_rows=77)
    assert bool((out[sum(rows):] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("single,prompt", [(200, 2048), (60, 4096), (300, 700)])
def test_a_prompt_next_to_single_tokens(code, single, prompt):
    """Single tokens of many sequences and a prompt in one call, through either kernel, appended and attended to."""
    rows = [1] * (single // 2) + [prompt] + [1] * (single - single // 2)
    lengths = [prompt + 5 if r > 1 else 1 + (37 * i) % 900 for i, r in enumerate(rows)]
    cache = Cache(lengths, 32, 2, 64, CODES[code], seed=single)
    _check_append(cache, rows, lengths, 2, torch.bfloat16, seed=1)
    _check_attend(cache, rows, lengths, 2, torch.bfloat16, seed=2)
