"""The paged 8-bit cache at its edges: scores far from zero. Tolerances as in test_kv_cache.py."""
import math

import pytest
import torch

import macko_spmv_b200 as macko_spmv
from test_kv_cache import CODES, TYPES, Cache, _attend_plain, _gen, _starts


def _check(cache, rows, lengths, q, scale=None, times=1):
    """`times`: the same sequences so many times over the same pages, so that there are units for all CTAs and none has to be cut."""
    lens = torch.tensor(lengths * times, dtype=torch.int32, device="cuda")
    table = cache.table.repeat(times, 1)
    out = macko_spmv.paged_attention(q.repeat(times, 1, 1), cache.tensors, table, lens, _starts(rows * times), scale)
    ref, weight, small = _attend_plain(q, cache, rows, lengths, scale if scale is not None else 1.0 / math.sqrt(cache.d))
    bound = (2.0 ** -11 + 2.0 ** -14) * weight + 2.0 ** -25 * small + torch.finfo(q.dtype).eps / 2 * ref.abs() * 1.01 + 2.0 ** -24
    off = (out.double().view(times, *ref.shape) - ref).abs()
    assert bool(((off <= bound) | (ref.isnan() & out.view(off.shape).isnan())).all()), float((off / bound).nan_to_num(1e30).max())


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
            _check(cache, rows, lengths, q.to(TYPES[dtype]))
