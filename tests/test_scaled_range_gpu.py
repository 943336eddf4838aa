"""Attention over the 8-bit cache with one scale for each (block, kv head) where the value scales of a context lie far apart: large
ones that a row gives no weight or does not see must not take bits from its result."""
import math

import pytest
import torch

from oracle import scaled_cache as oracle
from test_scaled_cache_gpu import DEV, KINDS, Cache, context, decode, half_ulp, random_query, tables_for

pytestmark = pytest.mark.gpu


def small_beside(c, query, tables, lens, new, scale, slopes=None, window=0, most=2.0 ** -4):
    """The tolerance would not pass a result that is lost: it is small against the rows' own largest elements."""
    row = 0
    for i, (n, total) in enumerate(zip(new, lens)):
        want, bound = oracle.attention(query[row:row + n].cpu(), c.key_codes, c.value_codes, c.key_scales, c.value_scales, tables[i], total,
                                       total - n, scale, c.kind, slopes, window)
        assert (bound.amax(2) <= most * want.abs().amax(2)).all()
        row += n


def check(got, c, query, tables, lens, new, scale, slopes=None, window=0):
    """check_attention, where results may also lie beyond the type's largest number (65504 of f16): those are infinities."""
    info = torch.finfo(query.dtype)
    row = 0
    for i, (n, total) in enumerate(zip(new, lens)):
        want, bound = oracle.attention(query[row:row + n].cpu(), c.key_codes, c.value_codes, c.key_scales, c.value_scales, tables[i], total,
                                       total - n, scale, c.kind, slopes, window)
        have = got[row:row + n].cpu().double()
        slack = bound + (want.abs() + bound) * half_ulp(query.dtype) + info.smallest_normal * info.eps
        inside = want.abs() <= info.max                        # (and there an infinity is as far off as the next number, 2^16)
        have = torch.where(have.isinf() & inside, torch.sign(have) * info.max * (1 + info.eps), have)
        assert not torch.isnan(have).any(), f"sequence {i}"
        off = torch.where(inside, (have - want).abs(), 0.0)
        assert (off <= slack).all(), f"sequence {i}: {float((off - slack).max())} over, {float((off / slack).max())} of it"
        beyond = want.abs() - slack > info.max
        assert (have[beyond] == torch.sign(want[beyond]) * math.inf).all(), f"sequence {i}: finite"
        row += n


def outlier(c, tables, at, ratio, u):
    """Block `at` of every sequence has value scales `ratio` times the others' and keys that look away from u [size]."""
    for b in tables[:, at].tolist():
        c.value_scales[b] *= ratio
        c.key_codes[b] = -torch.sign(u.double()) * 96
        c.key_scales[b] = 1.0
    c.upload()


def facing(u, rows, heads, dtype):
    """Queries that all lie along u, of several lengths."""
    return (u * torch.linspace(0.5, 1.0, rows * heads).view(rows, heads, 1)).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------ one new token
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,block,heads,kv_heads", [(128, 16, 8, 2), (64, 8, 2, 2), (80, 32, 6, 1), (256, 16, 4, 1)])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 17, 2.0 ** 26, 2.0 ** 60])
@pytest.mark.parametrize("parts", [1, 3])
def test_decode_a_large_scale_that_nobody_attends_to(kind, dtype, size, block, heads, kv_heads, ratio, parts):
    lens = [512, 2000]
    c = Cache(sum((n + block - 1) // block for n in lens) + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    u = torch.randn(size, generator=torch.Generator().manual_seed(5)).sign()
    outlier(c, tables, 9, ratio, u)
    query = facing(u, 2, heads, dtype)
    got = decode(c, query, tables, lens, 0.5 / size, parts=parts)
    small_beside(c, query, tables, lens, [1, 1], 0.5 / size)
    check(got, c, query, tables, lens, [1, 1], 0.5 / size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", [1, 4])
def test_decode_scales_against_scores(kind, parts):
    """Value scales that fall as fast as the weights rise, faster and slower."""
    lens = [700, 1500]
    c = Cache(150, 1, 128, 16, kind)
    tables = tables_for(lens, 16, 150)
    falling(c, tables)
    slopes = SLOPES
    query = random_query(2, 6, 128, torch.bfloat16) * 0.05
    got = decode(c, query, tables, lens, 0.09, slopes.to(DEV), parts)
    check(got, c, query, tables, lens, [1, 1], 0.09, slopes)


SLOPES = torch.tensor([0.0, 0.02, 0.0379, 0.0758, 0.1, 0.5])


def falling(c, tables):
    """A block's value scale is 2^-1.75 of the one before it, from 2^60 down: about exp(-0.0758) a token in blocks of 16; every ninth is 0."""
    for row in tables.tolist():
        for i, b in enumerate(x for x in row if x < len(c.value_scales)):
            c.value_scales[b] = 2.0 ** (60 - 1.75 * i) if i % 9 != 5 else 0.0
    c.upload()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_of_the_scale_zero_are_zeros(kind, dtype):
    """Whatever codes stand there, alone and beside others."""
    lens = [100, 300]
    c = Cache(30, 2, 128, 16, kind)
    tables = tables_for(lens, 16, 30)
    c.value_scales[tables[0, :7].long()] = 0
    c.value_scales[tables[1, ::3][tables[1, ::3] < 30].long()] = 0
    c.upload()
    query = random_query(2, 4, 128, dtype)
    got = decode(c, query, tables, lens, 0.09)
    assert (got[0] == 0).all()
    check(got, c, query, tables, lens, [1, 1], 0.09)
    query = random_query(130, 4, 128, dtype)
    for parts in (1, 2):
        got = context(c, query, tables, [0, 70], [70, 60], lens, 0.09, parts)
        assert (got[:70] == 0).all()
        check(got, c, query, tables, lens, [70, 60], 0.09)


# --------------------------------------------------------------------------------- several new tokens
SHAPES = [(128, 16, 8, 1), (128, 8, 4, 2), (64, 16, 4, 1), (80, 32, 5, 1), (112, 16, 4, 1), (256, 16, 4, 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 17, 2.0 ** 26, 2.0 ** 60])
@pytest.mark.parametrize("parts", [1, 3])
def test_context_a_large_scale_that_nobody_attends_to(kind, size, block, heads, kv_heads, ratio, parts):
    dtype = torch.bfloat16 if ratio > 2.0 ** 20 else torch.float16
    new, lens = [150, 3], [700, 330]
    c = Cache(sum((n + block - 1) // block for n in lens) + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    u = torch.randn(size, generator=torch.Generator().manual_seed(5)).sign()
    outlier(c, tables, 3, ratio, u)
    query = facing(u, 153, heads, dtype)
    got = context(c, query, tables, [0, 150], new, lens, 0.5 / size, parts)
    small_beside(c, query, tables, lens, new, 0.5 / size)
    check(got, c, query, tables, lens, new, 0.5 / size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("ratio", [2.0 ** 17, 2.0 ** 26, math.inf, math.nan])
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("window", [0, 70])
def test_context_rows_know_nothing_of_what_they_do_not_see(kind, size, block, heads, kv_heads, ratio, few, window):
    """The sequence's last block has a scale far above the others', or none at all: rows before it do as without it.  So do, with a
    window, rows behind a block that lies outside."""
    new, total = (6 if few else 140), 420 + 2 * block
    total = total // block * block + 2                           # two tokens in the last block
    c = Cache(total // block + 3, kv_heads, size, block, kind)
    tables = tables_for([total], block, c.key.shape[0])
    query = random_query(new, heads, size, torch.bfloat16)
    plain = context(c, query, tables, [0], [new], [total], 0.09, window=window)
    touched = [int(tables[0, total // block])] + ([int(tables[0, (total - new) // block - 2 - 70 // block])] if window else [])
    before = c.value_scales.clone()
    for b in touched:
        c.value_scales[b] *= ratio
    c.upload()
    got = context(c, query, tables, [0], [new], [total], 0.09, window=window)
    seen = new - 2
    # (a wave's sums may be brought to another power of two at another time: not the same bits)
    kept, c.value_scales = c.value_scales, before
    check(got[:seen], c, query[:seen], tables, [total - 2], [seen], 0.09, window=window)
    check(plain[:seen], c, query[:seen], tables, [total - 2], [seen], 0.09, window=window)
    c.value_scales = kept
    if math.isnan(ratio):
        assert got[seen:].isnan().all()
    if math.isfinite(ratio):
        check(got, c, query, tables, [total], [new], 0.09, window=window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("order", ["falling", "rising", "any"])
def test_context_scales_far_apart(kind, size, block, heads, kv_heads, parts, order):
    """Value scales that rise or fall by 2^7 a stage and by up to 2^60 a block, some zero."""
    new, lens = [140, 9], [900, 400]
    pages = sum((n + block - 1) // block for n in lens)
    c = Cache(pages + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    g = torch.Generator().manual_seed(8)
    for row, n in zip(tables.tolist(), lens):
        for i, b in enumerate(row[:(n + block - 1) // block]):
            power = {"falling": 40 - 7 * i * block / 64, "rising": -50 + 7 * i * block / 64}.get(order)
            c.value_scales[b] = 2.0 ** (int(torch.randint(-40, 20, (1,), generator=g)) if power is None else power)
            if i % 7 == 3:
                c.value_scales[b] = 0
    c.upload()
    slopes = torch.linspace(0, 0.15, heads)
    if order == "rising":
        slopes = -slopes
    query = random_query(149, heads, size, torch.bfloat16) * 0.1
    out = torch.full_like(query, 7.0)
    from splitwise_amd import _C
    _C.ops.context_attention_scaled(out, query, *c.device, 0.09, tables.to(DEV),
                                    *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 140], new, lens)), 140, 900,
                                    slopes.to(DEV), kind, num_parts=parts)
    small_beside(c, query, tables, lens, new, 0.09, slopes)
    check(out, c, query, tables, lens, new, 0.09, slopes)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("order", ["rising", "outlier"])
def test_context_tiles_of_256_rows(kind, order):
    """The launch of many workgroups: 64 heads of 128, of which a few are looked at."""
    heads, total, new = 64, 1150, 1100
    c = Cache(73, heads, 128, 16, kind)
    tables = tables_for([total], 16, 73)
    row = tables[0].long()
    if order == "rising":
        c.value_scales[row] = torch.exp2(-40 + 1.75 * torch.arange(72.0))[:, None].expand(-1, heads).contiguous()
        c.value_scales[row[11]] = 0
    else:
        c.value_scales[row[60]] *= 2.0 ** 26
    c.upload()
    some = [0, 13, 63]

    class Few:
        kind, key_codes, value_codes = c.kind, c.key_codes[:, :, some], c.value_codes[:, :, some]
        key_scales, value_scales = c.key_scales[:, some], c.value_scales[:, some]

    query = random_query(new, heads, 128, torch.bfloat16)
    got = context(c, query, tables, [0], [new], [total], 0.09)
    check(got[:, some], Few, query[:, some], tables, [total], [new], 0.09)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("power", [-100, 100])
@pytest.mark.parametrize("parts", [1, 3])
def test_all_scales_far_from_one(kind, size, block, heads, kv_heads, power, parts):
    """Of the few and of the many rows, next to each other and beside blocks of ordinary scales."""
    new, lens = [140, 3], [700, 330]
    c = Cache(sum((n + block - 1) // block for n in lens) + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    far = torch.exp2(power + torch.arange(float(len(c.value_scales))) % 5)[:, None]
    for some in (slice(None), slice(None, None, 2)):
        c.value_scales[some] = far[some].expand(-1, kv_heads)
        c.upload()
        query = random_query(143, heads, size, torch.bfloat16)
        got = context(c, query, tables, [0, 140], new, lens, 0.09, parts)
        check(got, c, query, tables, lens, new, 0.09)
        got = decode(c, query[:2], tables, lens, 0.09, parts=parts)
        check(got, c, query[:2], tables, lens, [1, 1], 0.09)
        c = Cache(len(c.value_scales), kv_heads, size, block, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40, 48, 100000])
@pytest.mark.parametrize("heads", [1, 8])
def test_windows_wider_than_any_context(kind, window, heads):
    """They hide nothing, also behind rows that stand before the sequence's first token."""
    new, lens = [70, 3], [40, 48]
    c = Cache(7, 1, 64, 16, kind)
    tables = tables_for(lens, 16, 7)
    query = random_query(73, heads, 64, torch.bfloat16)
    got = context(c, query, tables, [0, 70], new, lens, 0.1, window=window)
    assert torch.equal(got, context(c, query, tables, [0, 70], new, lens, 0.1))
    assert (got[:30] == 0).all()
    check(got, c, query, tables, lens, new, 0.1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("parts", [1, 3, None])
def test_attention_repeats_itself(kind, size, block, heads, kv_heads, parts):
    """The same bits from the same call, of few and of many rows, whatever the workspace held."""
    new, lens = [200, 5], [900, 330]
    c = Cache(sum((n + block - 1) // block for n in lens) + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    query = random_query(205, heads, size, torch.float16)
    few = [5, 5]
    first = [context(c, query, tables, [0, 200], new, lens, 0.09, parts), context(c, query, tables, [0, 5], few, lens, 0.09, parts),
             decode(c, query[:2], tables, lens, 0.09, parts=parts)]
    for _ in range(4):
        torch.empty(1 << 22, device=DEV).fill_(math.nan)
        again = [context(c, query, tables, [0, 200], new, lens, 0.09, parts), context(c, query, tables, [0, 5], few, lens, 0.09, parts),
                 decode(c, query[:2], tables, lens, 0.09, parts=parts)]
        assert all(torch.equal(a, b) for a, b in zip(first, again))
