"""The 8-bit cache with one scale for each (block, kv head) against 64 bits on the CPU (oracle/scaled_cache.py)."""
import math

import pytest
import torch

from oracle import scaled_cache as oracle
from splitwise_amd import _C

pytestmark = pytest.mark.gpu

KINDS = ["int8", "fp8_e4m3"]
DEV = "cuda"
U32 = 2.0 ** -24


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


class Cache:
    """A cache as earlier steps left it, on both sides; codes fill their range, no e4m3 NaN among them."""

    def __init__(self, blocks, heads, size, block, kind, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.block = kind, block
        top = oracle.TOP[kind]
        spread = torch.randn(blocks, block, 2 * heads, size, generator=g).double() * top / 3.4
        y = spread.clamp(-top, top)
        y = y.round() if kind == "int8" else y.float().to(torch.float8_e4m3fn).double()
        self.key_codes, self.value_codes = y[:, :, :heads].contiguous(), y[:, :, heads:].contiguous()
        self.key_scales = torch.exp(torch.randn(blocks, heads, generator=g) * 0.3) * 1.4 * 3.4 / top
        self.value_scales = torch.exp(torch.randn(blocks, heads, generator=g) * 0.6) * 3.4 / top
        self.upload()

    def upload(self):
        self.key = oracle.cache_of(self.key_codes, self.kind, True).to(DEV)
        self.value = oracle.cache_of(self.value_codes, self.kind, False).to(DEV)
        self.ks, self.vs = self.key_scales.to(DEV), self.value_scales.to(DEV)

    @property
    def device(self):
        return self.key, self.value, self.ks, self.vs


def tables_for(lens, block, blocks, seed=0, width=None):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(blocks, generator=g).tolist()
    pages = [(n + block - 1) // block for n in lens]
    assert sum(pages) <= blocks
    # what lies behind a sequence's blocks is never looked at
    t = torch.full((len(lens), width or max(1, max(pages))), 1 << 30, dtype=torch.int32)
    for i, p in enumerate(pages):
        t[i, :p] = torch.tensor(order[:p], dtype=torch.int32)
        order = order[p:]
    return t


def slots_of(tables, block, before, new):
    return torch.tensor([int(tables[i, t // block]) * block + t % block for i, (b, n) in enumerate(zip(before, new))
                         for t in range(b, b + n)], dtype=torch.int64)


# ------------------------------------------------------------------------------------------ write
def check_write(c, key, value, slots, seed=0):
    kind = c.kind
    _C.cache_ops.reshape_and_cache_scaled(key, value, *c.device, slots.to(DEV), kind)
    for name, x, cache, scales, codes, old in (("key", key, c.key, c.ks, c.key_codes, c.key_scales),
                                               ("value", value, c.value, c.vs, c.value_codes, c.value_scales)):
        new, want, touched = oracle.write(x.cpu(), codes, old, slots, kind)
        got_scales, got = scales.cpu().double(), oracle.codes_of(cache.cpu(), kind)
        rest = torch.ones(codes.shape[0], dtype=torch.bool)
        rest[touched] = False
        assert torch.equal(got[rest], codes[rest]) and torch.equal(got_scales[rest], old[rest].double()), f"{name}: untouched blocks"
        # amax * (1 / top): two roundings to 24 bits
        assert ((got_scales - new).abs() <= 2.1 * U32 * new).all(), f"{name}: scales"
        fresh = {s // c.block for s in slots.tolist() if s >= 0 and s % c.block == 0}
        written = {s for s in slots.tolist()}
        for b in touched:
            y = want[b].clone()
            if b in fresh:
                for o in range(c.block):
                    if b * c.block + o not in written:
                        y[o] = 0                              # a block that starts over is zeros elsewhere
            # the nearest code, of a quotient with four roundings (scale 2, reciprocal or ratio 1, product 1)
            slack = oracle.half_step(y.abs() * (1 + 2.0 ** -21), kind) + y.abs() * 4.1 * U32
            off = (got[b] - y).abs()
            assert (off <= slack).all(), f"{name}: block {b}, off {float((off - slack).max())}"
    return c


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,size,block", [(3, 64, 16), (2, 80, 8), (2, 96, 32), (1, 112, 16), (4, 128, 16), (3, 128, 32), (2, 128, 8),
                                              (2, 256, 16), (1, 256, 32)])
def test_write_prompts_and_tokens(kind, dtype, heads, size, block):
    """Whole blocks, the ends of prompts, chunks that begin inside a block, single tokens, padding; keys and values out of a fused
    projection."""
    c = Cache(40, heads, size, block, kind)
    before, new = [0, 5, 17, 40, 31, 64, 0], [3 * block, 1, 30, 1, 2 * block + 3, 1, 1]
    tables = tables_for([b + n for b, n in zip(before, new)], block, 40)
    slots = slots_of(tables, block, before, new)
    slots = torch.cat([slots[:40], torch.tensor([-1, -1]), slots[40:], torch.tensor([-1, 40 * block, 1 << 40])])
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(len(slots), 3 * heads * size, generator=g) * torch.exp(torch.randn(len(slots), 1, generator=g))
    qkv = qkv.to(dtype).to(DEV)
    key = qkv[:, heads * size:2 * heads * size].view(-1, heads, size)
    value = qkv[:, 2 * heads * size:].view(-1, heads, size)
    check_write(c, key, value, slots)


@pytest.mark.parametrize("kind", KINDS)
def test_write_many_tokens(kind):
    """The launch whose workgroups look at several entries of the list each."""
    c = Cache(110, 2, 64, 16, kind)
    before, new = [0, 3, 0, 0], [800, 400, 16, 7]
    slots = slots_of(tables_for([b + n for b, n in zip(before, new)], 16, 110), 16, before, new)
    key, value = (torch.randn(len(slots), 2, 64, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV) for i in (0, 1))
    check_write(c, key, value, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [37, 1100])
def test_write_in_any_order_and_twice(kind, count):
    """Tokens of one block anywhere in the list; of two for one slot the later one stays."""
    c = Cache(80, 2, 64, 16, kind)
    g = torch.Generator().manual_seed(count)
    slots = torch.randperm(80 * 16, generator=g)[:count]
    slots[count // 2] = slots[3]
    slots[count - 1] = slots[5]
    key, value = (torch.randn(count, 2, 64, generator=g).to(torch.float16).to(DEV) for _ in range(2))
    check_write(c, key, value, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_write_odd_values(kind, dtype):
    """Zeros, infinities, NaN, the types' largest and smallest values."""
    c = Cache(12, 1, 64, 16, kind)
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.randn(9 * 16, 1, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[:16] = 0
    x[16:32, 0, 3], x[16:32, 0, 4] = math.inf, -math.inf
    x[33, 0, 5] = math.nan
    x[48:64] = math.nan
    x[64:80] = math.inf
    x[81, 0, 0] = big
    x[96:112] = 0
    x[97, 0, 1] = tiny
    x[112:128] = -tiny
    slots = torch.arange(9 * 16)
    check_write(c, x.to(DEV), x.flip(0).contiguous().to(DEV), slots)


@pytest.mark.parametrize("kind", KINDS)
def test_write_one_token_at_a_time(kind):
    """A sequence that grows token by token through two blocks: each step is the oracle's step from what the last one left."""
    c = Cache(5, 2, 64, 16, kind)
    g = torch.Generator().manual_seed(2)
    for t in range(20):
        x = (torch.randn(1, 2, 64, generator=g) * (1 + t % 7)).to(torch.bfloat16)
        check_write(c, x.to(DEV), (-x).to(DEV), torch.tensor([32 + t]))
        c.key_codes, c.value_codes = oracle.codes_of(c.key.cpu(), kind), oracle.codes_of(c.value.cpu(), kind)
        c.key_scales, c.value_scales = c.ks.cpu(), c.vs.cpu()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [math.nan, math.inf, -1.0, 0.0])
def test_a_fresh_block_forgets(kind, scale):
    """A block that starts over takes nothing of what its memory held, NaN codes and odd scales included."""
    c = Cache(3, 1, 64, 16, kind)
    c.key.fill_(0x7f)
    c.value.fill_(0xff)
    c.ks.fill_(scale)
    c.vs.fill_(scale)
    x = torch.randn(3, 1, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    _C.cache_ops.reshape_and_cache_scaled(x, x, *c.device, torch.tensor([16, 17, 18], device=DEV), kind)
    for cache, scales in ((c.key, c.ks), (c.value, c.vs)):
        got = oracle.codes_of(cache.cpu(), kind)[1] * scales.cpu()[1].double()[:, None]
        assert (got[3:] == 0).all()
        assert (got[:3] - x.cpu().double()).abs().max() <= float(x.abs().max()) * (0.5 / 127 if kind == "int8" else 2.0 ** -4)


# ------------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,size,block", [(3, 64, 16), (2, 80, 8), (2, 96, 32), (1, 112, 16), (4, 128, 16), (2, 256, 32), (1, 256, 8)])
def test_read(kind, dtype, heads, size, block):
    lens = [0, 1, 3 * block, 50, 2 * block - 1, 0]
    c = Cache(60, heads, size, block, kind)
    tables = tables_for(lens, block, 60, width=20)
    starts = [2, 0, 70, 200, 4, 5]                            # (no rows shared: 4 + 63, 70 + 96)
    key = torch.full((262, 2 * heads, size), 7.0, dtype=dtype, device=DEV)[:, :heads]      # 250 ends the last row that is written
    value = torch.full((262, heads, size), 7.0, dtype=dtype, device=DEV)
    _C.cache_ops.gather_cache_scaled(key, value, *c.device, tables.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV),
                                     torch.tensor(lens, dtype=torch.int32, device=DEV), max(lens), kind)
    for got, codes, scales in ((key, c.key_codes, c.key_scales), (value, c.value_codes, c.value_scales)):
        want = torch.full((262, heads, size), 7.0, dtype=torch.float64)
        for i, n in enumerate(lens):
            if n:
                want[starts[i]:starts[i] + n] = oracle.rows(codes, scales, tables[i], n)[0]
        off = (got.cpu().double() - want).abs()
        # the product in 32 bits, the result in its type (or half a step of its smallest)
        assert (off <= want.abs() * (half_ulp(dtype) + 1.1 * U32) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()


@pytest.mark.parametrize("kind", KINDS)
def test_read_bounds(kind):
    """Lengths beyond the bound, the table or the output, and blocks that do not exist."""
    c = Cache(8, 2, 64, 16, kind)
    tables = torch.tensor([[0, 1, 2], [3, -1, 4], [5, 8, 6], [7, 7, 7]], dtype=torch.int32)
    lens, starts = [90, 40, 48, 48], [0, 50, 100, 150]
    out = [torch.full((160, 2, 64), 7.0, device=DEV) for _ in range(2)]
    _C.cache_ops.gather_cache_scaled(*out, *c.device, tables.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV),
                                     torch.tensor(lens, dtype=torch.int32, device=DEV), 1000, kind)
    for got, codes, scales in ((out[0], c.key_codes, c.key_scales), (out[1], c.value_codes, c.value_scales)):
        want = torch.full((160, 2, 64), 7.0, dtype=torch.float64)
        for i, n in enumerate([48, 40, 48, 10]):
            want[starts[i]:starts[i] + n] = oracle.rows(codes, scales, tables[i], n)[0]
        assert torch.equal(got.cpu(), want.float())


# -------------------------------------------------------------------------------------- attention
def check_attention(got, c, query, tables, lens, new, scale, slopes=None, window=0, decode=False, starts=None):
    dtype = query.dtype
    row = 0
    q = query.cpu()
    for i, (n, total) in enumerate(zip(new, lens)):
        if starts is not None:
            row = starts[i]
        want, bound = oracle.attention(q[row:row + n], c.key_codes, c.value_codes, c.key_scales, c.value_scales, tables[i], total,
                                       total - n, scale, c.kind, slopes, window)
        off = (got[row:row + n].cpu().double() - want).abs()
        slack = bound + (want.abs() + bound) * half_ulp(dtype) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert not torch.isnan(off).any(), f"sequence {i}"
        assert (off <= slack).all(), f"sequence {i}: {float((off - slack).max())} over, {float((off / slack).max())} of it"
        row += n


def random_query(rows, heads, size, dtype, seed=0):
    # rows out of a fused projection
    q = torch.randn(rows, heads + 2, size, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    return q[:, :heads]


LENS = [1, 0, 15, 16, 17, 63, 64, 65, 130, 257, 700]


def decode(c, query, tables, lens, scale, slopes=None, parts=None, most=None, out=None):
    out = torch.full_like(query, 7.0) if out is None else out
    _C.ops.paged_attention_scaled(out, query, *c.device, c.key.shape[1], scale, tables.to(DEV),
                                  torch.tensor(lens, dtype=torch.int32, device=DEV), c.block, max(lens) if most is None else most, slopes,
                                  c.kind, num_parts=parts)
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,size,block", [(4, 4, 64, 16), (6, 2, 80, 8), (4, 1, 96, 32), (2, 2, 112, 16), (16, 2, 128, 16),
                                                       (20, 1, 128, 16), (3, 1, 128, 32), (8, 2, 128, 8), (8, 2, 256, 16), (2, 1, 256, 32)])
@pytest.mark.parametrize("parts", [1, 3])
def test_decode(kind, dtype, heads, kv_heads, size, block, parts):
    c = Cache(sum((n + block - 1) // block for n in LENS) + 2, kv_heads, size, block, kind)
    tables = tables_for(LENS, block, c.key.shape[0])
    query = random_query(len(LENS), heads, size, dtype)
    got = decode(c, query, tables, LENS, size ** -0.5, parts=parts)
    check_attention(got, c, query, tables, LENS, [1 if n else 0 for n in LENS], size ** -0.5, starts=list(range(len(LENS))))
    assert (got[LENS.index(0)] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", [1, 2, 17, None])
def test_decode_slopes_and_parts(kind, parts):
    lens = [1500, 64, 1087, 3]
    c = Cache(170, 2, 64, 16, kind)
    tables = tables_for(lens, 16, 170)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.01, 0.003, 0.0])
    query = random_query(4, 6, 64, torch.bfloat16)
    got = decode(c, query, tables, lens, 0.2, slopes.to(DEV), parts)
    check_attention(got, c, query, tables, lens, [1] * 4, 0.2, slopes)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", [1, 4])
def test_decode_lengths_beyond_the_bound_are_done(kind, parts):
    """A bound that is too low costs time, not tokens."""
    lens = [700, 90]
    c = Cache(60, 1, 64, 16, kind)
    tables = tables_for(lens, 16, 60)
    query = random_query(2, 2, 64, torch.float16)
    check_attention(decode(c, query, tables, lens, 0.1, parts=parts, most=64), c, query, tables, lens, [1, 1], 0.1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("parts", [1, 2])
def test_decode_memory_that_holds_no_tokens(kind, block, parts):
    """NaN codes and NaN scales wherever no token is, blocks that do not exist, and tables that end before the length does."""
    lens = [37, 130, 5, 200, 90]
    c = Cache(80, 2, 128, block, kind)
    tables = tables_for(lens, block, 80)
    tables[3, 2], tables[3, 5] = -1, 80
    tables[4, :] = -3                                         # nothing of it exists
    used = torch.zeros(80, block, dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(n):
            if 0 <= int(tables[i, t // block]) < 80:
                used[int(tables[i, t // block]), t % block] = True
    nan = torch.full((), 0x7f, dtype=torch.uint8)
    for cache, axis in ((c.key, 3), (c.value, 3)):
        host = cache.cpu()
        mask = used[:, None, None, :, None] if cache.dim() == 5 else used[:, None, None, :]
        cache.copy_(torch.where(mask, host, nan))
    for scales in (c.ks, c.vs):
        scales[(~used.any(1)).to(DEV)] = math.nan
    query = random_query(5, 4, 128, torch.bfloat16)
    got = decode(c, query, tables, lens, 0.08, parts=parts)
    check_attention(got, c, query, tables, lens, [1] * 5, 0.08)
    assert (got[4] == 0).all()
    short = tables[:, :4].contiguous()                         # lengths are held to the table
    got = decode(c, query, short, lens, 0.08, parts=parts)
    check_attention(got, c, query, short, [min(n, 4 * block) for n in lens], [1] * 5, 0.08)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_far_apart_magnitudes(kind, dtype):
    """Value scales over many powers of two, some zero, queries at the ends of their type's range, scores that saturate the softmax."""
    lens = [300, 129, 64]
    c = Cache(40, 1, 128, 16, kind)
    g = torch.Generator().manual_seed(4)
    c.value_scales = torch.exp2(torch.randint(-60, 20, (40, 1), generator=g).float())
    c.value_scales[::5] = 0
    c.key_scales[::7] = 0
    c.upload()
    tables = tables_for(lens, 16, 40)
    query = random_query(3, 4, 128, torch.float32)
    size = [1e30, 1e-30, 1.0] if dtype == torch.bfloat16 else [400.0, 1e-4, 1.0]
    query = (query * torch.tensor(size, device=DEV)[:, None, None]).to(dtype)
    # (one scale for the call: the rows' scores are about 1e30 s, 1e-30 s and s)
    for scale, one in ((size[0] ** -1, 0), (size[1] ** -1, 1), (3.0, 2)):
        got = decode(c, query, tables, lens, scale)
        row, total = query[one:one + 1], lens[one]
        want, bound = oracle.attention(row.cpu(), c.key_codes, c.value_codes, c.key_scales, c.value_scales, tables[one], total, total - 1,
                                       scale, kind)
        off = (got[one].cpu().double() - want[0]).abs()
        finite = want[0].abs() < torch.finfo(dtype).max
        assert (off <= bound[0] + (want[0].abs() + bound[0]) * half_ulp(dtype) + 2.0 ** -24)[finite].all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,size,block", [(2, 2, 64, 16), (6, 2, 80, 8), (3, 1, 96, 32), (2, 2, 112, 16), (8, 1, 128, 16),
                                                       (5, 1, 128, 16), (4, 2, 128, 32), (4, 4, 128, 8), (2, 1, 256, 16), (20, 1, 64, 32)])
@pytest.mark.parametrize("window", [0, 40])
def test_context(kind, dtype, heads, kv_heads, size, block, window):
    new = [1, 5, 0, 33, 64, 130, 7, 17]
    lens = [1, 5, 40, 200, 64, 300, 257, 16]                   # (the last one has more new tokens than tokens: its first sees nothing)
    c = Cache(sum((n + block - 1) // block for n in lens) + 2, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    starts = [3, 4, 0, 9, 42, 110, 240, 250]
    query = random_query(270, heads, size, dtype)
    for parts in (1, 3):
        out = torch.full_like(query, 7.0)
        _C.ops.context_attention_scaled(out, query, *c.device, size ** -0.5, tables.to(DEV),
                                        *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (starts, new, lens)), max(new),
                                        max(lens), None, kind, sliding_window=window, num_parts=parts)
        check_attention(out, c, query, tables, lens, new, size ** -0.5, window=window, starts=starts)
        for i in (0, 1, 2, 106, 109, 247, 249, 267, 269):      # rows of no sequence
            assert (out[i] == 7.0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", [1, 2, None])
def test_context_long_with_slopes(kind, parts):
    """Many tiles of rows over many groups of tokens; rows that begin inside groups."""
    new, lens = [300, 77], [1111, 600]
    c = Cache(130, 2, 128, 16, kind)
    tables = tables_for(lens, 16, 130)
    slopes = torch.tensor([0.3, 0.02, 0.0, 0.001])
    query = random_query(377, 4, 128, torch.bfloat16)
    for window in (0, 100, 5000):
        out = torch.empty_like(query)
        _C.ops.context_attention_scaled(out, query, *c.device, 0.09, tables.to(DEV),
                                        *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 300], new, lens)), 300, 1111,
                                        slopes, kind, sliding_window=window, num_parts=parts)
        check_attention(out, c, query, tables, lens, new, 0.09, slopes, window)


@pytest.mark.parametrize("kind", KINDS)
def test_context_hidden_values(kind):
    """Blocks that do not exist, memory that holds no tokens, more new tokens than are asked for, rows behind the output."""
    new, lens = [70, 40], [150, 90]
    c = Cache(20, 1, 128, 16, kind)
    tables = tables_for(lens, 16, 20)
    tables[0, 1] = -1
    tables[1, 3] = 77
    tail = int(tables[0, 9])
    c.value[tail, :, :, 6:] = 0x7f
    c.key[tail, :, :, 6:] = 0x7f
    query = random_query(100, 2, 128, torch.bfloat16)
    args = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 70], new, lens)]
    out = torch.full_like(query, 7.0)
    _C.ops.context_attention_scaled(out, query, *c.device, 0.09, tables.to(DEV), *args, 70, 150, None, kind)
    padded = torch.cat([query, query[:10]])
    full = torch.full_like(padded, 7.0)
    _C.ops.context_attention_scaled(full, padded, *c.device, 0.09, tables.to(DEV), *args, 70, 150, None, kind)
    check_attention(full, c, padded, tables, lens, new, 0.09, starts=[0, 70])
    assert torch.equal(out, full[:100])
    few = torch.full_like(query, 7.0)
    _C.ops.context_attention_scaled(few, query, *c.device, 0.09, tables.to(DEV), *args, 33, 150, None, kind)
    check_attention(few[:33], c, query[:33], tables, [150 - 37], [33], 0.09)
    assert (few[33:70] == 7.0).all()


# ------------------------------------------------------------------------------------ used together
@pytest.mark.parametrize("kind", KINDS)
def test_a_conversation(kind):
    """A prompt, decode steps, a few drafted tokens, and reading it all back, as a serving loop strings them together; against the
    64-bit attention over what was read back."""
    block, heads, kv_heads, size = 16, 8, 2, 128
    lens = [45, 17, 80]
    c = Cache(30, kv_heads, size, block, kind)
    tables = tables_for([n + 12 for n in lens], block, 30)
    g = torch.Generator().manual_seed(9)

    def step(new):
        slots = slots_of(tables, block, lens, new).to(DEV)
        k, v = (torch.randn(sum(new), kv_heads, size, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
        _C.cache_ops.reshape_and_cache_scaled(k, v, *c.device, slots, kind)
        for i, n in enumerate(new):
            lens[i] += n
        c.key_codes, c.value_codes = oracle.codes_of(c.key.cpu(), kind), oracle.codes_of(c.value.cpu(), kind)
        c.key_scales, c.value_scales = c.ks.cpu(), c.vs.cpu()
        return torch.cat([k, v], 1)

    prompt, lens = lens, [0, 0, 0]
    first = step(prompt)
    for _ in range(5):
        step([1, 1, 1])
        query = random_query(3, heads, size, torch.bfloat16, seed=lens[0])
        check_attention(decode(c, query, tables, lens, 0.09), c, query, tables, lens, [1, 1, 1], 0.09)
    new = [4, 4, 4]
    step(new)
    query = random_query(12, heads, size, torch.bfloat16)
    out = torch.empty_like(query)
    _C.ops.context_attention_scaled(out, query, *c.device, 0.09, tables.to(DEV),
                                    *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 4, 8], new, lens)), 4, max(lens), None,
                                    kind)
    check_attention(out, c, query, tables, lens, new, 0.09)
    rows = [torch.empty(sum(prompt), kv_heads, size, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    starts = [0, prompt[0], prompt[0] + prompt[1]]
    _C.cache_ops.gather_cache_scaled(*rows, *c.device, tables.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV),
                                     torch.tensor(prompt, dtype=torch.int32, device=DEV), max(prompt), kind)
    got = torch.cat(rows, 1).float()
    # a block's largest value lies under 6 standard deviations; codes were rounded up to 6 times as its scale grew
    worst = 6 * 6 * (0.5 / 127 if kind == "int8" else 2.0 ** -4)
    assert (got - first.float()).abs().max() <= worst + 2.0 ** -8 * 6


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(kind):
    """A decode step in a graph: replays see new tokens, lengths and queries; eager work goes on between them."""
    block, heads, kv_heads, size = 16, 8, 2, 128
    c, twin = Cache(60, kv_heads, size, block, kind), Cache(60, kv_heads, size, block, kind)
    before = [400, 30]
    tables = tables_for([n + 8 for n in before], block, 60)
    on = dict(device=DEV)
    table = tables.to(DEV)
    slots, lens = torch.zeros(2, dtype=torch.int64, **on), torch.zeros(2, dtype=torch.int32, **on)
    x = torch.zeros(2, 2, kv_heads, size, dtype=torch.bfloat16, **on)
    query, out = (torch.zeros(2, heads, size, dtype=torch.bfloat16, **on) for _ in range(2))
    read = torch.zeros(2, 500, kv_heads, size, dtype=torch.bfloat16, **on)
    starts = torch.tensor([0, 450], dtype=torch.int32, **on)

    def step(c, out, read):
        _C.cache_ops.reshape_and_cache_scaled(x[0], x[1], *c.device, slots, kind)
        _C.ops.paged_attention_scaled(out, query, *c.device, kv_heads, 0.09, table, lens, block, 420, None, kind, num_parts=4)
        _C.cache_ops.gather_cache_scaled(read[0], read[1], *c.device, table, starts, lens, 420, kind)

    slots.copy_(slots_of(tables, block, before, [1, 1]))
    lens.copy_(torch.tensor([n + 1 for n in before]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in c.device]
    with torch.cuda.stream(side):
        step(c, out, read)
    torch.cuda.current_stream().wait_stream(side)
    for t, k in zip(c.device, keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):      # (as the workers capture: one process takes one kind)
        step(c, out, read)
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        x.copy_(torch.randn(x.shape, generator=g))
        query.copy_(torch.randn(query.shape, generator=g))
        at = [n + i for n in before]
        slots.copy_(slots_of(tables, block, at, [1, 1]))
        lens.copy_(torch.tensor([n + 1 for n in at]))
        graph.replay()
        torch.cuda.synchronize()
        eager, rows = torch.empty_like(out), torch.zeros_like(read)
        step(twin, eager, rows)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(read[:, :at[0] + 1], rows[:, :at[0] + 1])
        assert all(torch.equal(a, b) for a, b in zip(c.device, twin.device))


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(kind):
    """Split attention on two streams: each call has its own workspace."""
    c = Cache(70, 2, 64, 16, kind)
    tables = tables_for([500, 500], 16, 70)
    queries = [random_query(2, 4, 64, torch.float16, seed=i) for i in range(2)]
    want = [decode(c, q, tables, [500, 490], 0.1, parts=8) for q in queries]
    lens = torch.tensor([500, 490], dtype=torch.int32, device=DEV)
    table = tables.to(DEV)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(10)] for q in queries]
    for i in range(10):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                _C.ops.paged_attention_scaled(outs[j][i], queries[j], *c.device, 2, 0.1, table, lens, 16, 500, None, kind, num_parts=8)
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j]) for o in outs[j])


def test_results_repeat():
    """No order of atomics in them."""
    c = Cache(100, 2, 128, 16, "int8")
    tables = tables_for([1500], 16, 100)
    query = random_query(1, 16, 128, torch.bfloat16)
    first = decode(c, query, tables, [1500], 0.09)
    assert all(torch.equal(first, decode(c, query, tables, [1500], 0.09)) for _ in range(5))


def test_blocks_copy_and_swap_like_any_cache():
    """Codes and scales go through copy_blocks and swap_blocks (scales of 4 heads: 16 bytes a block)."""
    c = Cache(6, 4, 64, 16, "int8")
    _C.cache_ops.copy_blocks([c.key], [c.value], {1: [2, 3]})
    _C.cache_ops.copy_blocks([c.ks], [c.vs], {1: [2, 3]})
    for t in c.device:
        assert torch.equal(t[1], t[2]) and torch.equal(t[1], t[3])
    host = torch.empty(6, 4, dtype=torch.float32, pin_memory=True)
    _C.cache_ops.swap_blocks(c.ks, host, {3: 0})
    torch.cuda.synchronize()
    assert torch.equal(host[0], c.ks[3].cpu())


# --------------------------------------------------------------------------- the native side of small steps
@pytest.mark.parametrize("kind", KINDS)
def test_native_calls_do_the_same(kind, monkeypatch):
    """Each operator through the native host side and through Python: the same bits, and the native side takes the plain call."""
    from splitwise_amd import _native
    if isinstance(_native.step_ops, _native._NotBuilt):
        pytest.skip("_step_ops is not built")
    lens, new = [700, 33], [3, 2]
    tables = tables_for(lens, 16, 60).to(DEV)
    i32 = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 3], new, lens, [0, 700])]
    query = random_query(5, 4, 64, torch.bfloat16)
    x = random_query(5, 4, 64, torch.bfloat16, seed=1)
    slots = slots_of(tables.cpu(), 16, [a - b for a, b in zip(lens, new)], new).to(DEV)
    results = []
    for native in (True, False):
        answers = []

        class Seen:
            def __getattr__(self, name):
                def run(*args):
                    got = getattr(_native.step_ops, name)(*args) if native else None
                    answers.append(got)
                    return got
                return run

        monkeypatch.setattr(_C, "_native", Seen())
        c = Cache(60, 2, 64, 16, kind)
        _C.cache_ops.reshape_and_cache_scaled(x[:, :2], x[:, 2:], *c.device, slots, kind)
        rows = [torch.zeros(733, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
        _C.cache_ops.gather_cache_scaled(*rows, *c.device, tables, i32[3], i32[2], 700, kind)
        one = torch.empty_like(query[:2])
        _C.ops.paged_attention_scaled(one, query[:2], *c.device, 2, 0.1, tables, i32[2], 16, 700, None, kind)
        few = torch.empty_like(query)
        _C.ops.context_attention_scaled(few, query, *c.device, 0.1, tables, i32[0], i32[1], i32[2], 3, 700, None, kind, sliding_window=300)
        assert answers == [0 if native else None] * 4
        results.append([*c.device, *rows, one, few])
        with pytest.raises(RuntimeError, match="heads must be contiguous"):
            _C.ops.paged_attention_scaled(one, query[:2].transpose(1, 2), *c.device, 2, 0.1, tables, i32[2], 16, 700, None, kind)
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ------------------------------------------------------------------------- large, wide and repeated calls
def context(c, query, tables, starts, new, lens, scale, parts=None, out=None, window=None):
    out = torch.full_like(query, 7.0) if out is None else out
    _C.ops.context_attention_scaled(out, query, *c.device, scale, tables.to(DEV),
                                    *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (starts, new, lens)), max(new), max(lens),
                                    None, c.kind, sliding_window=window, num_parts=parts)
    return out


@pytest.mark.parametrize("kind", KINDS)
def test_a_cache_past_4_gib(kind):
    """Blocks on either side of 2^31 and 2^32 bytes and at the cache's end do as the same blocks of a small cache."""
    heads, size, block, total = 8, 128, 16, 266000             # 16 KiB a block: 4.06 GiB of keys and as much of values
    far = [0, 131071, 131072, 262143, 262144, 265998, 265999]
    lens = [40, 37]
    small = Cache(7, heads, size, block, kind)
    large = Cache(7, heads, size, block, kind)
    large.key, large.value = (torch.empty(total, *t.shape[1:], dtype=torch.uint8, device=DEV) for t in (small.key, small.value))
    large.ks, large.vs = (torch.zeros(total, heads, device=DEV) for _ in range(2))
    tables = torch.tensor([[6, 1, 3], [4, 2, 5]], dtype=torch.int32)
    wide = torch.full((2, 5), 1 << 30, dtype=torch.int32)      # rows of a wider table
    wide[:, 1:4] = torch.tensor(far, dtype=torch.int32)[tables.long()]
    g = torch.Generator().manual_seed(2)
    key, value = (torch.randn(sum(lens), heads, size, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    queries = random_query(sum(lens), 2 * heads, size, torch.bfloat16)
    results = []
    for c, t in ((small, tables), (large, wide[:, 1:4])):
        _C.cache_ops.reshape_and_cache_scaled(key, value, *c.device, slots_of(t, block, [0, 0], lens).to(DEV), kind)
        rows = [torch.zeros(77, heads, size, dtype=torch.float16, device=DEV) for _ in range(2)]
        table = torch.nn.functional.pad(t, (1, 1), value=1 << 30).to(DEV)[:, 1:4]
        i32 = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 40], lens)]
        _C.cache_ops.gather_cache_scaled(*rows, *c.device, table, *i32, 40, kind)
        outs = []
        for parts in (1, 2):
            outs.append(torch.empty_like(queries[:2]))
            _C.ops.paged_attention_scaled(outs[-1], queries[:2], *c.device, heads, 0.09, table, i32[1], block, 40, None, kind, num_parts=parts)
            outs.append(torch.empty_like(queries))
            _C.ops.context_attention_scaled(outs[-1], queries, *c.device, 0.09, table, i32[0], i32[1], i32[1], 40, 40, None, kind,
                                            num_parts=parts)
            # (rows by many: the kernel for long prompts)
            many = queries.repeat(1, 8, 1)
            outs.append(torch.empty_like(many))
            _C.ops.context_attention_scaled(outs[-1], many, *c.device, 0.09, table, i32[0], i32[1], i32[1], 40, 40, None, kind,
                                            num_parts=parts)
        results.append([*rows, *outs])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    check_write(Cache(7, heads, size, block, kind), key, value, slots_of(tables, block, [0, 0], lens))


def test_read_into_rows_far_apart():
    """A row of the output every 2^27 bytes, 5 GiB in all."""
    c = Cache(4, 2, 128, 16, "int8")
    step = 1 << 26
    buffer = torch.empty(39 * step + 2 * 128, dtype=torch.bfloat16, device=DEV)
    far = buffer.as_strided((40, 2, 128), (step, 128, 1))
    near = [torch.empty(40, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    args = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([[2, 0, 3]], [0], [40])]
    _C.cache_ops.gather_cache_scaled(near[0], near[1], *c.device, *args, 40, "int8")
    _C.cache_ops.gather_cache_scaled(near[2], far, *c.device, *args, 40, "int8")
    assert torch.equal(far, near[1]) and torch.equal(near[0], near[2])
    _C.cache_ops.gather_cache_scaled(far, near[2], *c.device, *args, 40, "int8")
    assert torch.equal(far, near[0]) and torch.equal(near[1], near[2])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,block", [(64, 16), (80, 8), (128, 16), (128, 32)])
def test_launches_of_many_workgroups(kind, size, block):
    """Shapes whose launches differ from the small ones': decode of many pairs, short prompts of many pairs by tiles of 16 rows, long ones
    by tiles of 256; the first and last sequences and a few heads are looked at."""
    kv_heads = 64
    lens = [1150, 40, 9] if block > 8 else [1150, 40]
    c = Cache(sum((n + block - 1) // block for n in lens) + 1, kv_heads, size, block, kind)
    tables = tables_for(lens, block, c.key.shape[0])
    some = [0, 13, 63]

    class Few:
        kind, key_codes, value_codes = c.kind, c.key_codes[:, :, some], c.value_codes[:, :, some]
        key_scales, value_scales = c.key_scales[:, some], c.value_scales[:, some]

    # one token each: 8 sequences of 64 heads, most of them the same
    pick = [1, 1, 1, 1, 1, 1, 1, len(lens) - 1]
    query = random_query(8, kv_heads, size, torch.float16)
    got = decode(c, query, tables[pick], [lens[i] for i in pick], size ** -0.5)
    check_attention(got[:, some], Few, query[:, some], tables[pick], [lens[i] for i in pick], [1] * 8, size ** -0.5)
    # 100 new tokens of 3 sequences, of which the short ones have fewer tokens than that
    pick = [0, 1, 1]
    query = random_query(300, kv_heads, size, torch.bfloat16)
    got = context(c, query, tables[pick], [0, 100, 200], [100, 30, 40], [1150, 40, 40], size ** -0.5)
    check_attention(got[:, some], Few, query[:, some], tables[pick], [1150, 40, 40], [100, 30, 40], size ** -0.5, starts=[0, 100, 200])
    # a whole prompt
    query = random_query(1150, kv_heads, size, torch.bfloat16)
    got = context(c, query, tables[:1], [0], [1140], [1150], size ** -0.5)
    check_attention(got[:, some], Few, query[:, some], tables[:1], [1150], [1140], size ** -0.5)
    assert (got[1140:] == 7.0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_scale_below_zero(kind, dtype):
    lens, new = [300, 70], [120, 3]
    c = Cache(30, 2, 64, 16, kind)
    tables = tables_for(lens, 16, 30)
    query = random_query(123, 4, 64, dtype)
    check_attention(context(c, query, tables, [0, 120], new, lens, -0.11), c, query, tables, lens, new, -0.11)
    check_attention(decode(c, query[:2], tables, lens, -0.11), c, query[:2], tables, lens, [1, 1], -0.11)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [4, 300])
def test_graphs_that_share_their_memory(kind, new):
    """Attention of several new tokens in two captured graphs of one pool, split and whole, replayed in turn with eager work between."""
    heads, kv_heads, size, block = 4, 2, 128, 16
    c = Cache(60, kv_heads, size, block, kind)
    tables = tables_for([800], block, 60).to(DEV)
    i32 = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(3)]
    query = torch.zeros(new, heads, size, dtype=torch.bfloat16, device=DEV)
    outs = [torch.zeros_like(query) for _ in range(3)]

    def run(out, parts):
        _C.ops.context_attention_scaled(out, query, *c.device, 0.09, tables, *i32, new, 800, None, kind, num_parts=parts)

    i32[1].fill_(new), i32[2].fill_(700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(outs[2], 1), run(outs[2], 3)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.inference_mode():
        with torch.cuda.graph(graphs[0]):
            run(outs[0], 3)
        with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
            run(outs[1], 1), run(outs[0], 2)
    for i in range(4):
        query.copy_(torch.randn(query.shape, generator=torch.Generator().manual_seed(i)))
        i32[2].fill_(520 + 90 * i)
        for which, (at, parts) in enumerate(((0, 3), (1, 1))):
            graphs[which].replay()
            torch.cuda.synchronize()
            run(outs[2], parts)
            assert torch.equal(outs[at], outs[2])
        run(outs[2], 2)
        assert torch.equal(outs[0], outs[2])
