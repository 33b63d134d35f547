"""The paged K/V cache entry points refuse what the host can check before any
device work, with a message, and leave no exception behind.  CPU."""
import ctypes as C
import importlib

import pytest


@pytest.fixture(scope="module")
def paged():
    return importlib.import_module("index-tts-25-metal_b200.paged")


@pytest.fixture(scope="module")
def lib(gpt_mod):
    return gpt_mod.load_library()


P = 0x10000  # an address that no refused call may touch


def tables(paged):
    return paged.Tables(4, 16, 100, 8, 8, 32, P, P, P, P, P, P, P, P, P, P, P)


def cache(paged, type=1, blocks=100, block=16, heads=2, dim=64):
    return paged.Cache(P, P, type, blocks, block, heads, dim, 0, block * heads * dim, heads * dim, dim,
                       block * heads * dim, heads * dim, dim)


def append(paged):
    return paged.Append(cache(paged), P, P, 1, 3, 128, 64, 128, 64, P)


def attention(paged):
    need = paged.workspace_bytes(64)
    return paged.Attention(cache(paged), P, 2 * P, 4, 3, 256, 64, 256, 64, P, P, P, 8, 4, 8, 1, 0.125, P, need)


def refused(lib, gpt_mod, entry, args, text):
    assert getattr(lib, entry)(0, C.byref(args), None) == gpt_mod.ERR_INVALID_ARGUMENT
    assert text in lib.itts_paged_last_error().decode()


@pytest.mark.parametrize("field,value,text", [
    ("requests", 0, "requests out of range"),
    ("requests", 8193, "requests out of range"),
    ("block_size", 24, "block_size is 16, 32, 64 or 128"),
    ("block_size", 256, "block_size is 16, 32, 64 or 128"),
    ("blocks", 0, "cache size out of range"),
    ("blocks", 1 << 27, "cache size out of range"),
    ("max_blocks", 0, "width out of range"),
    ("max_blocks", 1 << 27, "width out of range"),
    ("max_blocks", (1 << 26) + 1, "width out of range"),
    ("table_stride", 7, "stride out of range"),
    ("table_stride", 1 << 31, "stride out of range"),
    ("rows", -1, "rows out of range"),
    ("cached", None, "null argument"),
    ("fresh", None, "null argument"),
    ("table", None, "block table is null"),
    ("free_list", None, "null argument"),
    ("free_in", None, "null argument"),
    ("free_out", None, "null argument"),
    ("lens", None, "null argument"),
    ("q_start", None, "null argument"),
    ("positions", None, "null argument"),
    ("slots", None, "null argument"),
    ("status", None, "null argument"),
])
def test_tables_refusals(lib, gpt_mod, paged, field, value, text):
    a = tables(paged)
    setattr(a, field, value)
    refused(lib, gpt_mod, "itts_paged_tables", a, text)


CACHE_REFUSALS = [
    ("k", None, "cache is null"),
    ("v", None, "cache is null"),
    ("type", 3, "type is f32, f16 or bf16"),
    ("blocks", 0, "cache size out of range"),
    ("block_size", 8, "block_size is 16, 32, 64 or 128"),
    ("heads", 0, "heads out of range"),
    ("head_dim", 96, "head_dim is 64 or 128"),
    ("reserved", 1, "reserved"),
    ("k", P + 8, "multiples of 16 bytes"),
    ("v", P + 2, "multiples of 16 bytes"),
    ("k_token_stride", 132, "multiples of 16 bytes"),
    ("v_head_stride", 4, "multiples of 16 bytes"),
    ("k_block_stride", -2048, "multiples of 16 bytes"),
    ("v_block_stride", 1 << 39, "multiples of 16 bytes"),
]


@pytest.mark.parametrize("field,value,text", CACHE_REFUSALS)
def test_cache_refusals(lib, gpt_mod, paged, field, value, text):
    for make, entry in ((append, "itts_paged_append"), (attention, "itts_paged_attention")):
        a = make(paged)
        setattr(a.cache, field, value)
        refused(lib, gpt_mod, entry, a, text)


@pytest.mark.parametrize("field,value,text", [
    ("source_type", 2, "source type"),
    ("rows", -1, "rows out of range"),
    ("k", None, "null argument"),
    ("v", None, "null argument"),
    ("slots", None, "null argument"),
    ("k", P + 1, "misaligned"),
    ("v_row_stride", -1, "stride out of range"),
    ("k_head_stride", 1 << 40, "stride out of range"),
])
def test_append_refusals(lib, gpt_mod, paged, field, value, text):
    a = append(paged)
    setattr(a, field, value)
    refused(lib, gpt_mod, "itts_paged_append", a, text)


@pytest.mark.parametrize("field,value,text", [
    ("q", None, "null argument"),
    ("out", None, "null argument"),
    ("out", P, "must not overlap"),
    ("q", P + 8, "multiples of 16 bytes"),
    ("out_row_stride", 257, "multiples of 16 bytes"),
    ("q_heads", 3, "q_heads"),
    ("q_heads", 0, "q_heads"),
    ("q_heads", 258, "q_heads"),
    ("rows", -1, "rows out of range"),
    ("rows", (1 << 29) + 1, "rows out of range"),
    ("q_start", None, "null argument"),
    ("lens", None, "null argument"),
    ("table", None, "block table is null"),
    ("table_stride", 3, "stride out of range"),
    ("requests", 0, "requests out of range"),
    ("max_blocks", 0, "width out of range"),
    ("max_fresh", 0, "max_fresh"),
    ("scale", float("nan"), "scale must be finite"),
    ("scale", float("inf"), "scale must be finite"),
    ("workspace", None, "workspace"),
    ("workspace", P + 16, "workspace"),
    ("workspace_bytes", 255, "workspace"),
])
def test_attention_refusals(lib, gpt_mod, paged, field, value, text):
    a = attention(paged)
    setattr(a, field, value)
    refused(lib, gpt_mod, "itts_paged_attention", a, text)


def test_null_args_and_sizes(lib, gpt_mod, paged):
    for entry in ("itts_paged_tables", "itts_paged_append", "itts_paged_attention"):
        assert getattr(lib, entry)(0, None, None) == gpt_mod.ERR_INVALID_ARGUMENT
        assert "args is null" in lib.itts_paged_last_error().decode()
    assert paged.workspace_bytes(96) == 0
    assert paged.workspace_bytes(64) > 0 and paged.workspace_bytes(128) >= paged.workspace_bytes(64)


def test_qwen_batch_needs_a_context(lib, gpt_mod):
    assert lib.itts_qwen_generate_batch(None, 0, None, None, 8, None, None, None) == gpt_mod.ERR_INVALID_ARGUMENT


def test_no_rows_is_no_work(lib, gpt_mod, paged):
    a = append(paged)
    a.rows = 0
    assert lib.itts_paged_append(0, C.byref(a), None) == gpt_mod.OK
    b = attention(paged)
    b.rows = 0
    assert lib.itts_paged_attention(0, C.byref(b), None) == gpt_mod.OK


def test_packed_arguments_match_the_structs(paged):
    """paged.py packs the argument structs by hand: byte for byte what the ctypes classes hold."""
    for pack, kind in ((paged._PACK_TABLES, paged.Tables), (paged._PACK_APPEND, paged.Append),
                       (paged._PACK_ATTENTION, paged.Attention)):
        def flat(cls):
            for _, t in cls._fields_:
                yield from flat(t) if hasattr(t, "_fields_") else [t]

        values = [0.5 if t is C.c_float else 1000003 * (i + 1) for i, t in enumerate(flat(kind))]
        it = iter(values)

        def build(cls):
            return cls(*[build(t) if hasattr(t, "_fields_") else next(it) for _, t in cls._fields_])

        assert bytes(build(kind)) == pack(*values)


def test_python_binding_refuses_host_tensors(gpt_mod, paged):
    import torch
    i = torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(1, 2, 64)
    c = torch.zeros(3, 16, 2, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.append(x, x, c, c, i)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.attention(x, c, c, i[None], i, i, 1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.tables(i, i, i[None], i, i, 16, lens=i, q_start=i, positions=i, slots=i, status=i)


@pytest.mark.parametrize("field", ["k_block_stride", "k_token_stride", "k_head_stride", "v_block_stride", "v_token_stride",
                                   "v_head_stride"])
def test_append_refuses_a_repeated_dimension(lib, gpt_mod, paged, field):
    a = append(paged)
    setattr(a.cache, field, 0)
    refused(lib, gpt_mod, "itts_paged_append", a, "repeats a dimension")


@pytest.mark.parametrize("field", ["out_row_stride", "out_head_stride"])
def test_attention_refuses_a_repeated_output(lib, gpt_mod, paged, field):
    a = attention(paged)
    setattr(a, field, 0)
    refused(lib, gpt_mod, "itts_paged_attention", a, "out repeats a dimension")
