"""The 8-bit cache with one scale for each (block, kv head): refusals, which need no GPU, and the oracle's own consistency."""
import ctypes

import pytest
import torch

from oracle import scaled_cache as oracle
from splitwise_amd import _C

BLOCKS, HEADS, SIZE, BLOCK = 6, 2, 64, 16


def caches(blocks=BLOCKS, heads=HEADS, size=SIZE, block=BLOCK):
    return (torch.zeros(blocks, heads, size // 16, block, 16, dtype=torch.uint8), torch.zeros(blocks, heads, size, block, dtype=torch.uint8),
            torch.zeros(blocks, heads), torch.zeros(blocks, heads))


def write(key=None, value=None, cache=None, slots=None, kind="int8"):
    key = torch.zeros(3, HEADS, SIZE) if key is None else key
    value = torch.zeros_like(key) if value is None else value
    _C.cache_ops.reshape_and_cache_scaled(key, value, *(cache or caches()), torch.arange(3) if slots is None else slots, kind)


@pytest.mark.parametrize("kind", ["auto", "fp8_e5m2", "int4"])
def test_other_cache_types_are_refused(kind):
    with pytest.raises(RuntimeError, match="Unsupported data type of kv cache"):
        write(kind=kind)


def test_write_refuses_what_it_would_misread():
    k, v, ks, vs = caches()
    for bad, why in [(dict(cache=(k.to(torch.int16), v, ks, vs)), "uint8"), (dict(cache=(k, v, ks.double(), vs)), "float32"),
                     (dict(cache=(k, v[0], ks, vs)), "value cache"), (dict(cache=(k[:, :, :2], v, ks, vs)), "key cache"),
                     (dict(cache=(k, v, ks[:3], vs)), "scales"), (dict(cache=(k, v, ks, vs.t().contiguous().t())), "contiguous"),
                     (dict(cache=caches(heads=4)), "key cache"), (dict(slots=torch.arange(4)), "slot_mapping"),
                     (dict(slots=torch.arange(3, dtype=torch.int32)), "slot_mapping"),
                     (dict(value=torch.zeros(3, HEADS, SIZE, dtype=torch.bfloat16)), "one shape and type"),
                     (dict(value=torch.zeros(2, HEADS, SIZE)), "one shape and type"),
                     (dict(key=torch.zeros(3, SIZE, HEADS).transpose(1, 2)), "heads must be contiguous")]:
        with pytest.raises(RuntimeError, match=why):
            write(**bad)
    with pytest.raises(RuntimeError, match="HIP device"):
        write()


def read(tables=None, starts=None, lens=None, rows=torch.zeros(5, HEADS, SIZE)):
    tables = torch.zeros(2, 3, dtype=torch.int32) if tables is None else tables
    starts = torch.zeros(2, dtype=torch.int32) if starts is None else starts
    lens = torch.zeros(2, dtype=torch.int32) if lens is None else lens
    _C.cache_ops.gather_cache_scaled(rows, torch.zeros_like(rows), *caches(), tables, starts, lens, 5, "fp8_e4m3")


def test_read_refuses_what_it_would_misread():
    for bad, why in [(dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
                     (dict(tables=torch.zeros(2, 6, dtype=torch.int32)[:, ::2]), "block_tables"),
                     (dict(tables=torch.zeros(3, 3, dtype=torch.int32)), "starts and lengths"),
                     (dict(starts=torch.zeros(2, dtype=torch.int64)), "starts and lengths"),
                     (dict(lens=torch.zeros(4, dtype=torch.int32)[::2]), "starts and lengths")]:
        with pytest.raises(RuntimeError, match=why):
            read(**bad)
    with pytest.raises(RuntimeError, match="HIP device"):
        read()


def attend(query=torch.zeros(2, 4, SIZE, dtype=torch.float16), out=None, kv_heads=HEADS, block=BLOCK, slopes=None, tables=None,
           context=False):
    out = torch.zeros_like(query) if out is None else out
    tables = torch.zeros(2, 3, dtype=torch.int32) if tables is None else tables
    lens = torch.ones(2, dtype=torch.int32)
    if context:
        _C.ops.context_attention_scaled(out, query, *caches(), 0.1, tables, lens * 0, lens, lens, 1, 1, slopes, "int8")
    else:
        _C.ops.paged_attention_scaled(out, query, *caches(), kv_heads, 0.1, tables, lens, block, 1, slopes, "int8")


def test_attention_refuses_what_it_would_misread():
    q = torch.zeros(2, 4, SIZE)
    for bad, why in [(dict(query=q), "Unsupported data type"), (dict(out=q.bfloat16()), "one shape and type"),
                     (dict(slopes=torch.zeros(3)), "alibi_slopes"), (dict(slopes=torch.zeros(4).double()), "alibi_slopes")]:
        for context in (False, True):
            with pytest.raises(RuntimeError, match=why):
                attend(context=context, **bad)
    with pytest.raises(RuntimeError, match="key cache"):
        attend(kv_heads=4)
    with pytest.raises(RuntimeError, match="blocks of 16 tokens"):
        attend(block=32)
    with pytest.raises(RuntimeError, match="one row of block_tables"):
        attend(tables=torch.zeros(3, 3, dtype=torch.int32))
    for context in (False, True):
        with pytest.raises(RuntimeError, match="HIP device"):
            attend(context=context)


def entry_point(name, **changed):
    """The entry point's status for plain arguments but those given; nothing it refuses is launched."""
    p = ctypes.c_void_p(1 << 20)
    common = dict(out=p, query=p, key_cache=p, value_cache=p, key_scales=p, value_scales=p, num_seqs=2, num_heads=4, num_kv_heads=2,
                  head_size=64, scale=0.1, block_tables=p, block_size=16, num_blocks=6, max_context_len=30, max_blocks_per_seq=3,
                  table_stride=3, alibi_slopes=None, q_stride=256, out_stride=256, act_dtype=_C.SW_F16, cache_dtype=_C.SW_I8_SCALED,
                  num_parts=1, workspace=None, workspace_bytes=0, stream=None)
    rows = dict(key=p, value=p, key_cache=p, value_cache=p, key_scales=p, value_scales=p, num_heads=2, head_size=64, block_size=16,
                num_blocks=6, key_stride=128, value_stride=128, act_dtype=_C.SW_F32, cache_dtype=_C.SW_E4M3_SCALED, stream=None)
    order = {
        "sw_paged_attention_scaled": (common | dict(context_lens=p), "out query key_cache value_cache key_scales value_scales num_seqs "
                                      "num_heads num_kv_heads head_size scale block_tables context_lens block_size num_blocks "
                                      "max_context_len max_blocks_per_seq table_stride alibi_slopes q_stride out_stride act_dtype "
                                      "cache_dtype num_parts workspace workspace_bytes stream"),
        "sw_context_attention_scaled": (common | dict(num_rows=4, seq_starts=p, new_lens=p, seq_lens=p, max_new_len=2, sliding_window=0),
                                        "out query key_cache value_cache key_scales value_scales num_seqs num_rows num_heads "
                                        "num_kv_heads head_size scale block_tables seq_starts new_lens seq_lens block_size num_blocks "
                                        "max_new_len max_context_len max_blocks_per_seq table_stride alibi_slopes sliding_window "
                                        "q_stride out_stride act_dtype cache_dtype num_parts workspace workspace_bytes stream"),
        "sw_reshape_and_cache_scaled": (rows | dict(slot_mapping=p, num_tokens=3), "key value key_cache value_cache key_scales "
                                        "value_scales slot_mapping num_tokens num_heads head_size block_size num_blocks key_stride "
                                        "value_stride act_dtype cache_dtype stream"),
        "sw_gather_cache_scaled": (rows | dict(block_tables=p, seq_starts=p, seq_lens=p, num_seqs=2, max_seq_len=20, num_rows=5,
                                               max_blocks_per_seq=3, table_stride=3),
                                   "key value key_cache value_cache key_scales value_scales block_tables seq_starts seq_lens num_seqs "
                                   "max_seq_len num_rows num_heads head_size block_size num_blocks max_blocks_per_seq table_stride "
                                   "key_stride value_stride act_dtype cache_dtype stream"),
    }
    values, names = order[name]
    assert not set(changed) - set(names.split())
    lib = _C.load_library()
    return getattr(lib, name)(*[{**values, **changed}[n] for n in names.split()]), lib.sw_last_error().decode()


ODD = ctypes.c_void_p((1 << 20) + 8)


@pytest.mark.parametrize("name,changed,why", [
    (n, c, w) for n in ("sw_paged_attention_scaled", "sw_context_attention_scaled") for c, w in [
        (dict(head_size=72), "head size"), (dict(block_size=64), "block size"), (dict(num_heads=5), "query heads"),
        (dict(num_kv_heads=0), "query heads"), (dict(num_blocks=0), "blocks"), (dict(num_blocks=1 << 31), "blocks"),
        (dict(num_seqs=-1), "sequences"), (dict(num_seqs=1 << 16), "sequences"), (dict(act_dtype=_C.SW_F32), "f16 and bf16"),
        (dict(cache_dtype=_C.SW_FP8_E5M2), "cache type"), (dict(query=ODD), "16 bytes"), (dict(out=ODD), "16 bytes"),
        (dict(q_stride=132), "16 bytes"), (dict(key_cache=ODD), "16 bytes"), (dict(num_parts=0), "parts"),
        (dict(num_parts=2), "workspace"), (dict(num_parts=2, workspace=ctypes.c_void_p(1 << 20), workspace_bytes=64), "workspace"),
        (dict(max_blocks_per_seq=1 << 27), "too wide"), (dict(max_context_len=-1), "negative")]
] + [("sw_context_attention_scaled", dict(max_new_len=1 << 30), "new tokens"),
     ("sw_context_attention_scaled", dict(num_rows=-1), "negative")] + [
    (n, c, w) for n in ("sw_reshape_and_cache_scaled", "sw_gather_cache_scaled") for c, w in [
        (dict(head_size=48), "head size"), (dict(block_size=4), "block size"), (dict(act_dtype=_C.SW_FP8_E5M2), "activation type"),
        (dict(cache_dtype=_C.SW_F16), "cache type"), (dict(key=ODD), "16 bytes"), (dict(value_stride=130), "16 bytes"),
        (dict(value_cache=ODD), "16 bytes"), (dict(num_heads=0), "heads"), (dict(num_blocks=-1), "blocks")]
] + [("sw_reshape_and_cache_scaled", dict(num_tokens=-1), "tokens"), ("sw_gather_cache_scaled", dict(num_seqs=1 << 16), "sequences"),
     ("sw_gather_cache_scaled", dict(max_seq_len=-1), "negative")])
def test_entry_points_refuse_before_a_launch(name, changed, why):
    status, message = entry_point(name, **changed)
    assert status == -1 and why in message, message


@pytest.mark.parametrize("name,changed,why", [
    ("sw_reshape_and_cache_scaled", dict(num_tokens=(1 << 31) - 1, num_heads=256), "too many"),
    ("sw_gather_cache_scaled", dict(max_seq_len=(1 << 31) - 1, max_blocks_per_seq=1 << 27, num_heads=2), "too long"),
    ("sw_gather_cache_scaled", dict(value_stride=1 << 26), "2^28 bytes"),
    ("sw_context_attention_scaled", dict(max_new_len=1 << 24), "new tokens")])
def test_launches_that_no_grid_holds_are_refused(name, changed, why):
    status, message = entry_point(name, **changed)
    assert status == -1 and why in message, message


@pytest.mark.parametrize("name,changed", [
    ("sw_paged_attention_scaled", dict(num_seqs=0)), ("sw_context_attention_scaled", dict(num_rows=0)),
    ("sw_context_attention_scaled", dict(max_new_len=0)), ("sw_reshape_and_cache_scaled", dict(num_tokens=0)),
    ("sw_gather_cache_scaled", dict(num_seqs=0)), ("sw_gather_cache_scaled", dict(max_blocks_per_seq=0)),
    ("sw_gather_cache_scaled", dict(num_rows=0))])
def test_calls_with_nothing_to_do_launch_nothing(name, changed):
    assert entry_point(name, **changed)[0] == 0


def test_parts_fill_the_chip_and_no_more():
    lib = _C.load_library()
    assert lib.sw_scaled_attention_parts(256, 1, 32, 32, 128, 4000) == 1
    assert lib.sw_scaled_attention_parts(1, 1, 64, 8, 128, 100) == 1
    assert 1 < lib.sw_scaled_attention_parts(1, 1, 64, 8, 128, 100000) <= 1024
    assert lib.sw_scaled_attention_workspace_bytes(1, 5, 4, 64) == 0
    assert lib.sw_scaled_attention_workspace_bytes(3, 5, 4, 64) == 3 * 5 * 4 * 68 * 4


@pytest.mark.parametrize("kind", ["int8", "fp8_e4m3"])
def test_oracle_codes_go_both_ways(kind):
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(0, 256, (3, 2, 4, 8, 16), dtype=torch.uint8, generator=g)
    raw[(raw & 127) == 127] = 0                              # e4m3's NaN
    raw[raw == 128] = 0                                      # its negative zero
    assert torch.equal(oracle.cache_of(oracle.codes_of(raw, kind), kind, True), raw)
    raw = raw.view(3, 2, 64, 8)
    assert torch.equal(oracle.cache_of(oracle.codes_of(raw, kind), kind, False), raw)


# ------------------------------------------------------------------------------------------- engine options
def test_engine_options_that_a_cache_with_scales_excludes():
    from splitwise_amd.config import CacheConfig
    from splitwise_amd.engine.arg_utils import EngineArgs
    for kind in ("int8", "fp8_e4m3"):
        assert CacheConfig(16, 0.9, 0, kind, enable_prefix_caching=True).cache_dtype == kind
        with pytest.raises(NotImplementedError, match="sliding window"):
            CacheConfig(16, 0.9, 0, kind, sliding_window=64)
        for more in (dict(sep_prompt_token=True), dict(overlap_prompt_decode=True, pipeline_steps=True)):
            with pytest.raises(NotImplementedError, match="scales"):
                EngineArgs(model="llama-tiny", kv_cache_dtype=kind, **more).create_engine_configs()
    with pytest.raises(NotImplementedError, match="prefix caching"):
        CacheConfig(16, 0.9, 0, "fp8_e5m2", enable_prefix_caching=True)
    with pytest.raises(ValueError, match="Unknown kv cache dtype"):
        CacheConfig(16, 0.9, 0, "int4")


def test_scales_count_in_a_block():
    import types
    from splitwise_amd.worker.cache_engine import CacheEngine
    model = types.SimpleNamespace(dtype=torch.bfloat16, get_head_size=lambda: 64, get_num_layers=lambda p: 3, get_num_kv_heads=lambda p: 2)
    size = lambda kind: CacheEngine.get_cache_block_size(16, kind, model, None)  # noqa: E731
    assert size("auto") == 3 * 2 * 16 * 2 * 64 * 2 and size("fp8_e5m2") == size("auto") // 2
    assert size("int8") == size("fp8_e4m3") == size("fp8_e5m2") + 3 * 2 * 2 * 4


def test_every_kernel_that_is_built_is_launched():
    """Workgroups of eight waves exist for heads of 80 to 128, which the launch rule gives them to, and for no others."""
    import re
    with open(_C.library_path(), "rb") as f:
        names = set(re.findall(rb"scaled_context_kernelILb([01])ELi(\d+)ELi(\d+)ELi(\d+)E", f.read()))
    built = {(int(e), int(head), int(block), int(waves)) for e, head, block, waves in names}
    assert built == {(e, head, block, waves) for e in (0, 1) for block in (8, 16, 32) for waves in (4, 8)
                     for head in ((64, 80, 96, 112, 128, 256) if waves == 4 else (80, 96, 112, 128))}


def test_workspace_of_a_long_list():
    """None for lists that are gone through; a number for each block and one more for others.  What is too small is refused."""
    lib = _C.load_library()
    size = lib.sw_reshape_and_cache_scaled_indexed_workspace_bytes
    assert size(0, 6) == size(1, 6) == size(256, 1 << 20) == 0
    assert size(5000, 6) == 28 and size(5000, (1 << 31) - 1) == 1 << 33
    p = ctypes.c_void_p(1 << 20)
    for work, nbytes in ((p, 24), (ctypes.c_void_p((1 << 20) + 2), 28)):
        status = lib.sw_reshape_and_cache_scaled_indexed(p, p, p, p, p, p, p, 5000, 2, 64, 16, 6, 128, 128, _C.SW_F32, _C.SW_E4M3_SCALED, work,
                                                         nbytes, None)
        assert status == -1 and "workspace" in lib.sw_last_error().decode()


def test_blocks_of_odd_bytes_are_not_copied():
    lib = _C.load_library()
    p = ctypes.c_void_p(1 << 20)
    for nbytes in (2, 6, 17, 0, -4):
        assert lib.sw_copy_blocks(p, p, 1, p, 1, nbytes, None) == -1 and "block_bytes" in lib.sw_last_error().decode()


def test_the_reason_of_a_refused_option_is_its_own():
    """Only pools of several workers have a transport: the option that runs both sides on one worker is not refused for it."""
    from splitwise_amd.engine.arg_utils import EngineArgs
    with pytest.raises(NotImplementedError) as told:
        EngineArgs(model="llama-tiny", kv_cache_dtype="int8", overlap_prompt_decode=True, pipeline_steps=True).create_engine_configs()
    text = str(told.value)
    assert "overlap_prompt_decode, whose two streams" in text and "sep_prompt_token, as the transport" in text


@pytest.mark.parametrize("kind", ["int8", "fp8_e4m3"])
def test_models_of_32_bits_are_refused_before_they_are_loaded(kind):
    from splitwise_amd.engine.arg_utils import EngineArgs
    with pytest.raises(NotImplementedError, match="float16 and bfloat16"):
        EngineArgs(model="llama-tiny", dtype="float32", kv_cache_dtype=kind).create_engine_configs()
    for dtype in ("auto", "float16", "bfloat16"):
        EngineArgs(model="llama-tiny", dtype=dtype, kv_cache_dtype=kind).create_engine_configs()
    EngineArgs(model="llama-tiny", dtype="float32", kv_cache_dtype="fp8_e5m2").create_engine_configs()
