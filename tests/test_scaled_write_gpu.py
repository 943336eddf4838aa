"""Writing the 8-bit cache with one scale for each (block, kv head): lists that name blocks and slots more than once."""
import random

import pytest
import torch

from test_scaled_cache_gpu import DEV, KINDS, Cache, check_write

pytestmark = pytest.mark.gpu


def fill(block, b):
    return [b * block + i for i in range(block)]


def written(kind, block, slots, heads=3, size=64, blocks=200, dtype=torch.bfloat16):
    c = Cache(blocks, heads, size, block, kind)
    g = torch.Generator().manual_seed(len(slots))
    key, value = (torch.randn(len(slots), heads, size, generator=g) * torch.exp(torch.randn(len(slots), 1, 1, generator=g)) for _ in "kv")
    check_write(c, key.to(dtype).to(DEV), value.to(dtype).to(DEV), torch.tensor(slots))


def padding(block, long):
    """What makes the list a long one: blocks that it fills, and some single tokens."""
    return [s for b in range(60, 60 + 1100 // block) for s in fill(block, b)] + [3 + 55 * block] if long else []


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("case", ["behind", "before", "around", "twice", "thrice and one", "right before", "right behind", "two runs of half",
                                  "far before", "one slot often", "one run, its own order"])
def test_a_run_that_fills_its_block_and_others_of_it(kind, block, long, case):
    f, other, more = fill(block, 2), fill(block, 4), padding(block, long)
    half = block // 2
    slots = {
        "behind": f + other + more + [f[3]],
        "before": [f[0], f[5]] + other + more + f,
        "around": [f[1]] + other + f + more + [f[block - 1], other[0]],
        "twice": f + more + other + f,
        "thrice and one": f + other + f + more + [f[2]] + other + f,
        "right before": other + [f[4]] + f + more,
        "right behind": other + f + [f[0]] + more,
        "two runs of half": f[:half] + other + more + f[half:],
        "far before": [f[7]] + more + other + f + other,
        "one run, its own order": [f[5], f[3], f[3], f[0], f[5]] + more + other[::-1],
        "one slot often": [f[2]] * 5 + more + [f[2]] + f + [f[6]] * 3,
    }[case]
    written(kind, block, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seed", range(6))
def test_lists_of_anything(kind, seed):
    """Runs that fill blocks, pieces of runs, single tokens, padding, of few blocks many times, in any order."""
    rng = random.Random(seed)
    block = rng.choice([8, 16, 32])
    blocks = rng.choice([12, 60])
    slots = []
    while len(slots) < rng.choice([200, 900, 1500, 4000]):
        f = fill(block, rng.randrange(blocks))
        how = rng.random()
        if how < 0.5:
            slots += f
        elif how < 0.7:
            a = rng.randrange(block)
            slots += f[a:a + rng.randint(1, block)]
        elif how < 0.9:
            slots += [rng.choice(f)]
        else:
            slots += [-1, blocks * block + 5 if blocks * block + 5 >= 200 * block else -7]
    written(kind, block, slots, dtype=rng.choice([torch.bfloat16, torch.float16, torch.float32]))


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_list_gives_the_same_cache(kind):
    """Whatever the order in which workgroups run: 2000 entries of 9 blocks."""
    rng = random.Random(1)
    slots = torch.tensor([s for _ in range(120) for s in (fill(16, rng.randrange(9)) if rng.random() < 0.6 else [rng.randrange(144)])])
    x = torch.randn(2, len(slots), 8, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    from splitwise_amd import _C
    first = None
    for _ in range(6):
        c = Cache(9, 8, 128, 16, kind)
        _C.cache_ops.reshape_and_cache_scaled(x[0], x[1], *c.device, slots.to(DEV), kind)
        first = first or [t.clone() for t in c.device]
        assert all(torch.equal(a, b) for a, b in zip(first, c.device))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seed", range(3))
def test_without_a_workspace(kind, seed, monkeypatch):
    """The entry point that takes none writes the same cache from any list, short and long."""
    from splitwise_amd import _C
    lib = _C.load_library()
    rng = random.Random(seed)
    for count in (300, 1500):
        slots = torch.tensor([s for _ in range(count) for s in (fill(16, rng.randrange(12)) if rng.random() < 0.1 else
                                                                [rng.randrange(192)])][:count])
        x = torch.randn(2, count, 3, 64, generator=torch.Generator().manual_seed(seed)).to(torch.float16).to(DEV)
        a, b = Cache(12, 3, 64, 16, kind), Cache(12, 3, 64, 16, kind)
        on = slots.to(DEV)
        _C.cache_ops.reshape_and_cache_scaled(x[0], x[1], *a.device, on, kind)
        assert lib.sw_reshape_and_cache_scaled(x[0].data_ptr(), x[1].data_ptr(), *(t.data_ptr() for t in b.device), on.data_ptr(), count, 3, 64,
                                               16, 12, 192, 192, _C.SW_F16, _C._SCALED[kind], torch.cuda.current_stream().cuda_stream) == 0
        assert all(torch.equal(p, q) for p, q in zip(a.device, b.device))


@pytest.mark.parametrize("kind", KINDS)
def test_long_lists_in_graphs_that_share_their_memory(kind):
    """Two captured writes of one pool, replayed in turn with eager work between; lists whose blocks have one run, and others."""
    from splitwise_amd import _C
    count, blocks = 1600, 120
    g = torch.Generator().manual_seed(4)
    slots = torch.zeros(2, count, dtype=torch.int64, device=DEV)
    x = torch.zeros(2, 2, count, 2, 64, dtype=torch.bfloat16, device=DEV)
    caches = [Cache(blocks, 2, 64, 16, kind, seed=i) for i in range(2)]
    twins = [Cache(blocks, 2, 64, 16, kind, seed=i) for i in range(2)]

    def run(c, i):
        _C.cache_ops.reshape_and_cache_scaled(x[i, 0], x[i, 1], *c.device, slots[i], kind)

    slots.fill_(-1)                                            # (nothing is written while the graphs are made)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(caches[0], 0)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.inference_mode():
        for i in range(2):
            with torch.cuda.graph(graphs[i], **({} if i == 0 else {"pool": graphs[0].pool()})):
                run(caches[i], i)
    for turn in range(4):
        for i in range(2):
            order = torch.randperm(blocks, generator=g)[:100]
            one = (order[:, None] * 16 + torch.arange(16)).flatten()
            if (turn + i) % 2:
                one[torch.randint(0, count, (40,), generator=g)] = one[torch.randint(0, count, (40,), generator=g)]
            slots[i].copy_(one)
            x[i].copy_(torch.randn(x[i].shape, generator=g))
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            run(twins[i], i)
            assert all(torch.equal(a, b) for a, b in zip(caches[i].device, twins[i].device))


@pytest.mark.parametrize("heads", [1, 2, 3, 4, 5, 8, 40])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_scales_of_any_number_of_heads_are_copied(heads, offset):
    """A block's scales are 4 bytes a head: blocks of no multiple of 16 bytes begin on 4; those of other blocks stay."""
    from splitwise_amd import _C
    offset = 4 * offset if heads % 4 == 0 else offset
    some = [torch.rand(7 * heads + offset, device=DEV)[offset:].view(7, heads) for _ in range(6)]
    before = [t.clone() for t in some]
    _C.cache_ops.copy_blocks(some[:3], some[3:], {1: [2, 3], 5: [6]})
    for now, was in zip(some, before):
        assert torch.equal(now, was[[0, 1, 1, 1, 4, 5, 5]])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [1e-45, 1e-39, 2.0 ** -127, 2.0 ** -111])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_scale_that_no_write_leaves_is_none(kind, scale, dtype):
    """Zeros, and then numbers, for a block that was never written and whose memory holds a scale without a finite reciprocal."""
    from oracle import scaled_cache as oracle
    from splitwise_amd import _C
    c = Cache(3, 2, 64, 16, kind)
    c.ks.fill_(scale), c.vs.fill_(scale)
    x = torch.zeros(1, 2, 64, dtype=dtype, device=DEV)
    slot = torch.tensor([16 + 3], device=DEV)
    _C.cache_ops.reshape_and_cache_scaled(x, x, *c.device, slot, kind)
    for cache, scales in ((c.key, c.ks), (c.value, c.vs)):
        assert (oracle.codes_of(cache.cpu(), kind)[1] == 0).all() and (scales[1] == 0).all()
    x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    _C.cache_ops.reshape_and_cache_scaled(x, x, *c.device, slot, kind)
    for cache, scales in ((c.key, c.ks), (c.value, c.vs)):
        got = oracle.codes_of(cache.cpu(), kind)[1] * scales.cpu()[1].double()[:, None]
        assert (got[torch.arange(16) != 3] == 0).all()
        assert (got[3] - x[0].cpu().double()).abs().max() <= float(x.abs().max()) * (0.51 / 127 if kind == "int8" else 2.0 ** -4)
