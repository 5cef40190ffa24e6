"""What the grouped-query operators refuse before anything is launched: by the torch layer on tensors without storage, by the C entry
points on made-up pointers that are never read."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from dscuda_b200 import flash, library

BF16, F32, I32, I8, U8 = torch.bfloat16, torch.float32, torch.int32, torch.int8, torch.uint8
B, T, HQ, HKV, PAGE, BLOCKS, PAGES = 2, 3, 8, 2, 32, 7, 4
MISSING = "[Dd]river|data pointer|storage|[Nn]o CUDA|NVIDIA"


def fake(*shape, dtype=BF16, device="cuda:0"):
    with FakeTensorMode():
        return torch.empty(shape, dtype=dtype, device=device)


def wider(*shape, by=2):
    """Rows that lie apart: a part of a fused projection."""
    with FakeTensorMode():
        return torch.empty(*shape[:-2], shape[-2] * by, shape[-1], dtype=BF16, device="cuda:0")[..., : shape[-2], :]


def rope(query=None, key=None, positions=None, sections=(16, 24, 24), **given):
    return flash.rope(fake(B, T, HQ, 128) if query is None else query, fake(B, T, HKV, 128) if key is None else key,
                      fake(len(sections), B, T, dtype=I32) if positions is None else positions, sections, **given)


def append(**given):
    x = dict(key_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=I8), value_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=I8), key_scale=fake(BLOCKS, HKV, dtype=F32),
             value_scale=fake(BLOCKS, HKV, dtype=F32), key=fake(B, T, HKV, 128), value=fake(B, T, HKV, 128), block_table=fake(B, PAGES, dtype=I32),
             start_positions=fake(B, dtype=I32), token_counts=fake(B, dtype=I32))
    return flash.cache_append(**{**x, **given})


def decode(**given):
    x = dict(query=fake(B, T, HQ, 128), key_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=I8), value_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=I8),
             key_scale=fake(BLOCKS, HKV, dtype=F32), value_scale=fake(BLOCKS, HKV, dtype=F32), block_table=fake(B, PAGES, dtype=I32),
             cache_lengths=fake(B, dtype=I32), scale=0.1)
    return flash.decode(**{**x, **given})


def cross(**given):
    x = dict(query=fake(B, 50, HQ, 128), key=fake(B, 70, HKV, 128), value=fake(B, 70, HKV, 128), scale=0.1, key_lengths=fake(B, dtype=I32))
    return flash.cross_forward(**{**x, **given})


def cross_back(**given):
    x = dict(dout=fake(B, 50, HQ, 128), output=fake(B, 50, HQ, 128), lse=fake(B, HQ, 50, dtype=F32), query=fake(B, 50, HQ, 128), key=fake(B, 70, HKV, 128),
             value=fake(B, 70, HKV, 128), scale=0.1, key_lengths=fake(B, dtype=I32))
    return flash.cross_backward(**{**x, **given})


DECODE_BYTES = library.library("flash_attention").dscuda_flash_decode_workspace_bytes(B, T, HQ, HKV)
BACK_BYTES = library.library("flash_attention").dscuda_flash_cross_backward_workspace_bytes(B, 50, 70, HQ, HKV)

REFUSED = {
    "rope_dtype": lambda: rope(query=fake(B, T, HQ, 128, dtype=torch.float16)),
    "rope_other_tokens": lambda: rope(key=fake(B, T + 1, HKV, 128)),
    "rope_other_width": lambda: rope(key=fake(B, T, HKV, 64)),
    "rope_other_device": lambda: rope(key=fake(B, T, HKV, 128, device="cuda:1")),
    "rope_positions_dtype": lambda: rope(positions=fake(3, B, T, dtype=torch.int64)),
    "rope_positions_axes": lambda: rope(positions=fake(2, B, T, dtype=I32)),
    "rope_positions_tokens": lambda: rope(positions=fake(3, B, T - 1, dtype=I32)),
    "rope_positions_device": lambda: rope(positions=fake(3, B, T, dtype=I32, device="cuda:1")),
    "rope_nothing": lambda: flash.rope(None, None, fake(1, T, dtype=I32), (64,)),
    "rope_empty": lambda: rope(query=fake(B, 0, HQ, 128)),
    "rope_output_without_input": lambda: flash.rope(fake(T, HQ, 128), None, fake(1, T, dtype=I32), (64,), key_out=fake(T, HQ, 128)),
    "rope_output_shape": lambda: rope(query_out=fake(B, T, HQ + 1, 128)),
    "rope_output_dtype": lambda: rope(query_out=fake(B, T, HQ, 128, dtype=F32)),
    "rope_output_device": lambda: rope(key_out=fake(B, T, HKV, 128, device="cuda:1")),
    "rope_heads_apart": lambda: rope(query=fake(B, T, HQ, 256)[..., :128]),
    "rope_tokens_unevenly_apart": lambda: rope(query=fake(B, T + 2, HQ, 128)[:, :T]),
    "append_dtype": lambda: append(key=fake(B, T, HKV, 128, dtype=F32)),
    "append_cache_dtype": lambda: append(key_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=U8)),
    "append_caches_differ": lambda: append(value_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=torch.float8_e4m3fn)),
    "append_cache_shapes_differ": lambda: append(value_cache=fake(BLOCKS - 1, HKV, PAGE, 128, dtype=I8)),
    "append_scale_dtype": lambda: append(key_scale=fake(BLOCKS, HKV, dtype=BF16)),
    "append_scale_shape": lambda: append(value_scale=fake(BLOCKS, HKV, PAGE, dtype=F32)),
    "append_scale_device": lambda: append(value_scale=fake(BLOCKS, HKV, dtype=F32, device="cuda:1")),
    "append_heads": lambda: append(key=fake(B, T, HKV + 1, 128), value=fake(B, T, HKV + 1, 128)),
    "append_value_tokens": lambda: append(value=fake(B, T + 1, HKV, 128)),
    "append_table_batch": lambda: append(block_table=fake(B + 1, PAGES, dtype=I32)),
    "append_table_dtype": lambda: append(block_table=fake(B, PAGES, dtype=torch.int64)),
    "append_starts": lambda: append(start_positions=fake(B - 1, dtype=I32)),
    "append_counts_dtype": lambda: append(token_counts=fake(B, dtype=torch.int64)),
    "append_three_dimensions": lambda: append(key=fake(B * T, HKV, 128)),
    "decode_heads_of_the_cache": lambda: decode(key_scale=fake(BLOCKS, HKV + 1, dtype=F32)),
    "decode_width": lambda: decode(query=fake(B, T, HQ, 64)),
    "decode_dtype": lambda: decode(query=fake(B, T, HQ, 128, dtype=torch.float16)),
    "decode_lengths": lambda: decode(cache_lengths=fake(B + 1, dtype=I32)),
    "decode_lengths_dtype": lambda: decode(cache_lengths=fake(B, dtype=torch.int64)),
    "decode_table_batch": lambda: decode(block_table=fake(B - 1, PAGES, dtype=I32)),
    "decode_query_device": lambda: decode(query=fake(B, T, HQ, 128, device="cuda:1")),
    "decode_query_strided": lambda: decode(query=wider(B, T, HQ, 128)),
    "decode_workspace": lambda: decode(workspace=fake(DECODE_BYTES - 1, dtype=U8)),
    "decode_workspace_device": lambda: decode(workspace=fake(DECODE_BYTES, dtype=U8, device="cuda:1")),
    "decode_output": lambda: decode(output=fake(B * T * HQ * 128 - 1)),
    "decode_lse": lambda: decode(lse=fake(B * T * HQ - 1, dtype=F32)),
    "cross_key_batch": lambda: cross(key=fake(B + 1, 70, HKV, 128)),
    "cross_value_keys": lambda: cross(value=fake(B, 71, HKV, 128)),
    "cross_width": lambda: cross(key=fake(B, 70, HKV, 64), value=fake(B, 70, HKV, 64)),
    "cross_lengths": lambda: cross(key_lengths=fake(B, 1, dtype=I32)),
    "cross_lengths_device": lambda: cross(key_lengths=fake(B, dtype=I32, device="cuda:1")),
    "cross_output": lambda: cross(output=fake(B, 49, HQ, 128)),
    "cross_few_rows_workspace": lambda: cross(query=fake(B, 1, HQ, 128), workspace=fake(16, dtype=U8)),
    "back_dout": lambda: cross_back(dout=fake(B, 49, HQ, 128)),
    "back_output_dtype": lambda: cross_back(output=fake(B, 50, HQ, 128, dtype=F32)),
    "back_lse": lambda: cross_back(lse=fake(B, 50, HQ, dtype=F32)),
    "back_workspace": lambda: cross_back(workspace=fake(BACK_BYTES - 1, dtype=U8)),
    "back_two_gradients": lambda: cross_back(grads=[fake(B, 50, HQ, 128), fake(B, 70, HKV, 128)]),
    "back_gradient_size": lambda: cross_back(grads=[fake(B, 50, HQ, 128), fake(B, 69, HKV, 128), fake(B, 70, HKV, 128)]),
    "back_gradient_dtype": lambda: cross_back(grads=[fake(B, 50, HQ, 128, dtype=F32), fake(B, 70, HKV, 128), fake(B, 70, HKV, 128)]),
}


@pytest.mark.parametrize("call", REFUSED.values(), ids=REFUSED.keys())
def test_refused(call):
    with pytest.raises(ValueError):
        call()


ACCEPTED = {
    "rope": lambda: rope(),
    "rope_rows": lambda: flash.rope(fake(T, HQ, 64), None, fake(2, T, dtype=I32), (8, 24)),
    "rope_part_of_a_projection": lambda: rope(query=wider(B, T, HQ, 128), key=wider(B, T, HKV, 128, by=5)),
    "rope_given": lambda: rope(query_out=wider(B, T, HQ, 128), key_out=fake(B, T, HKV, 128)),
    "append": lambda: append(),
    "append_part_of_a_projection": lambda: append(key=wider(B, T, HKV, 128), value=wider(B, T, HKV, 128)),
    "append_no_starts": lambda: append(start_positions=None, token_counts=None),
    "append_e4m3": lambda: append(key_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=torch.float8_e4m3fn), value_cache=fake(BLOCKS, HKV, PAGE, 128, dtype=torch.float8_e4m3fn)),
    "decode": lambda: decode(),
    "decode_given": lambda: decode(workspace=fake(DECODE_BYTES // 4 + 1, dtype=F32), output=fake(B, T, HQ, 128), lse=fake(B, HQ, T, dtype=F32)),
    "cross": lambda: cross(),
    "cross_all_keys": lambda: cross(key_lengths=None),
    "cross_single_token": lambda: cross(query=fake(B, 1, HQ, 128)),
    "cross_backward": lambda: cross_back(grads=[fake(B, 50, HQ, 128), fake(B, 70, HKV, 128), fake(B, 70, HKV, 128)], workspace=fake(BACK_BYTES, dtype=U8)),
}


@pytest.mark.parametrize("call", ACCEPTED.values(), ids=ACCEPTED.keys())
def test_what_fits_is_accepted(call):
    """The call gets past the checks: what ends it is the missing storage or, without a driver, the device."""
    with pytest.raises(RuntimeError, match=MISSING):
        call()


@pytest.mark.parametrize("call", [
    lambda: flash.rope(torch.zeros(T, HQ, 128, dtype=BF16), None, torch.zeros(1, T, dtype=I32), (64,)),
    lambda: append(key=torch.zeros(B, T, HKV, 128, dtype=BF16)),
    lambda: decode(cache_lengths=torch.zeros(B, dtype=I32)),
    lambda: cross(key=torch.zeros(B, 70, HKV, 128, dtype=BF16)),
    lambda: cross_back(lse=torch.zeros(B, HQ, 50)),
], ids=["rope", "append", "decode", "cross", "backward"])
def test_host_memory_is_refused(call):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()


# ---- the C entry points: addresses that are aligned, or not, and never read ----------------------------------------

AT = 4096


def refused(name, *arguments):
    lib = library.library("flash_attention")
    assert getattr(lib, "dscuda_flash_" + name)(*arguments) == 1
    return lib.dscuda_flash_last_error().decode()


def c_rope(query_out=AT, key_out=AT, query=AT, key=AT, positions=AT, rows=4, hq=8, hk=2, width=128, strides=(1024, 256, 1024, 256), sections=(16, 24, 24), theta=10000.0,
           axes=None, none=False):
    array = (ctypes.c_int * len(sections))(*sections)
    return refused("rope", query_out, key_out, query, key, positions, rows, hq, hk, width, *strides, len(sections) if axes is None else axes,
                   None if none else array, 0, 0, theta, None)


@pytest.mark.parametrize("given,message", [
    (dict(width=96), "head_size 64 or 128"), (dict(query_out=None), "null"), (dict(query=None, query_out=None, key=None, key_out=None), "null"),
    (dict(positions=None), "null"), (dict(rows=0), "positive rows"), (dict(hq=0), "positive rows"), (dict(hk=-1), "positive rows"), (dict(hq=70000), "positive rows"),
    (dict(theta=1.0), "theta > 1"), (dict(theta=float("nan")), "theta > 1"), (dict(theta=float("inf")), "theta > 1"), (dict(sections=(64, 0)), "add up"),
    (dict(sections=(32, 31)), "add up"), (dict(sections=(60, 70, -66)), "add up"), (dict(sections=(16,) * 4, axes=5), "one to four"), (dict(axes=0), "one to four"),
    (dict(none=True), "one to four"), (dict(strides=(1024, 256, 1023, 256)), "16 bytes"), (dict(strides=(1024, 248, 1024, 256)), "overlap"),
    (dict(strides=(2048, 256, 1024, 256)), "in place"), (dict(query=AT + 2), "16-byte"), (dict(positions=AT + 2), "4-byte"),
])
def test_rope_entry_point(given, message):
    assert message in c_rope(**given)


def c_append(pointers=(AT,) * 9, batch=2, tokens=3, heads=2, width=128, strides=(256, 256), page=32, pages=4, blocks=7, kind=0):
    return refused("cache_append", *pointers, batch, tokens, heads, width, *strides, page, pages, blocks, kind, None)


def replaced(count, at, value):
    return (AT,) * at + (value,) + (AT,) * (count - at - 1)


@pytest.mark.parametrize("given,message", [
    (dict(width=64), "head_size 128"), (dict(kind=2), "int8 or e4m3"), (dict(batch=0), "positive batch"), (dict(tokens=0), "positive batch"), (dict(heads=-2), "positive batch"),
    (dict(pages=0), "positive batch"), (dict(blocks=0), "positive batch"), (dict(page=24), "multiple of 16"), (dict(page=0), "multiple of 16"),
    (dict(page=1 << 16, pages=1 << 15), "index range"), (dict(blocks=1 << 30, page=64), "index range"), (dict(batch=70000), "index range"), (dict(heads=40000, strides=(1 << 23,) * 2), "index range"),
    (dict(strides=(248, 256)), "overlap"), (dict(strides=(256, 260)), "16 bytes"), (dict(pointers=replaced(9, 0, None)), "null"), (dict(pointers=replaced(9, 2, None)), "null"),
    (dict(pointers=replaced(9, 1, AT + 8)), "16-byte"), (dict(pointers=replaced(9, 5, AT + 2)), "16-byte"), (dict(pointers=replaced(9, 6, None)), "null"),
    (dict(pointers=replaced(9, 7, AT + 1)), "4-byte"),
])
def test_append_entry_point(given, message):
    assert message in c_append(**given)


def c_decode(pointers=(AT,) * 10, missing=0, batch=2, tokens=3, hq=8, hkv=2, width=128, page=32, pages=4, blocks=7, kind=0, scale=0.1):
    size = library.library("flash_attention").dscuda_flash_decode_workspace_bytes(batch, tokens, hq, hkv)
    return refused("decode", *pointers, max(0, size - missing), batch, tokens, hq, hkv, width, page, pages, blocks, kind, scale, None)


@pytest.mark.parametrize("given,message", [
    (dict(width=64), "head_size 128"), (dict(kind=-1), "int8 or e4m3"), (dict(hq=9), "divisible"), (dict(hq=0), "divisible"), (dict(hkv=0), "positive batch"),
    (dict(tokens=65), "at most 64"), (dict(tokens=0), "positive batch"), (dict(scale=0.0), "positive softmax scale"), (dict(scale=float("nan")), "positive softmax scale"),
    (dict(batch=70000), "index range"), (dict(hq=5000, hkv=1), "4096"), (dict(missing=1), "too small"), (dict(pointers=replaced(10, 9, None)), "null"),
    (dict(pointers=replaced(10, 2, AT + 4)), "16-byte"), (dict(pointers=replaced(10, 1, AT + 2)), "4-byte"), (dict(pointers=replaced(10, 8, None)), "null"),
    (dict(batch=60000, page=1 << 20, pages=1 << 10, blocks=2, hkv=2, hq=8), "index range"),
])
def test_decode_entry_point(given, message):
    assert message in c_decode(**given)


def c_cross(pointers=(AT,) * 7, missing=0, batch=2, tq=50, tk=70, hq=8, hkv=2, width=128, scale=0.1):
    size = library.library("flash_attention").dscuda_flash_cross_forward_workspace_bytes(batch, tq, tk, hq, hkv)
    return refused("cross_forward", *pointers, max(0, size - missing), batch, tq, tk, hq, hkv, width, scale, None)


def c_cross_back(pointers=(AT,) * 11, missing=0, batch=2, tq=50, tk=70, hq=8, hkv=2, width=128, scale=0.1):
    size = library.library("flash_attention").dscuda_flash_cross_backward_workspace_bytes(batch, tq, tk, hq, hkv)
    return refused("cross_backward", *pointers, max(0, size - missing), batch, tq, tk, hq, hkv, width, scale, None)


@pytest.mark.parametrize("call", [c_cross, c_cross_back])
@pytest.mark.parametrize("given,message", [
    (dict(width=64), "head_size 128"), (dict(tq=0), "positive batch"), (dict(tk=0), "positive batch"), (dict(batch=-1), "positive batch"), (dict(hq=9), "divisible"),
    (dict(hkv=0), "divisible"), (dict(hq=130), "at most 64"), (dict(scale=-0.1), "positive softmax scale"), (dict(batch=70000), "index range"),
    (dict(batch=4, tk=1 << 30), "index range"), (dict(tq=1 << 28, hq=16), "index range"),
])
def test_cross_entry_points(call, given, message):
    assert message in call(**given)


@pytest.mark.parametrize("call,given,message", [
    (c_cross, dict(tq=1, missing=1), "too small"), (c_cross, dict(pointers=replaced(7, 6, None), tq=1), "null"), (c_cross, dict(pointers=replaced(7, 0, None)), "null"),
    (c_cross, dict(pointers=replaced(7, 3, AT + 8)), "16-byte"), (c_cross, dict(pointers=replaced(7, 5, AT + 2)), "4-byte"),
    (c_cross_back, dict(missing=1), "too small"), (c_cross_back, dict(pointers=replaced(11, 1, AT + 2)), "16-byte"), (c_cross_back, dict(pointers=replaced(11, 5, None)), "null"),
    (c_cross_back, dict(pointers=replaced(11, 10, None)), "null"),
])
def test_cross_pointers(call, given, message):
    assert message in call(**given)


@pytest.mark.parametrize("shape", [(0, 1, 8, 2), (1, 0, 8, 2), (1, 1, 0, 2), (1, 1, 8, 0), (-1, -1, -1, -1)])
def test_size_queries_survive_empty_shapes(shape):
    lib = library.library("flash_attention")
    assert lib.dscuda_flash_decode_workspace_bytes(*shape) == 0
    assert lib.dscuda_flash_cross_forward_workspace_bytes(shape[0], shape[1], 5, *shape[2:]) == 0
    assert lib.dscuda_flash_cross_backward_workspace_bytes(shape[0], shape[1], 5, *shape[2:]) == 0


def test_workspace_sizes():
    """Parts of at most 444 CTAs, two each, of 8, 16 or 32 rows, and 8 bytes for each entry, head and block of rows."""
    lib = library.library("flash_attention")
    for batch, tokens, hq, hkv in ((1, 1, 32, 8), (32, 1, 32, 8), (8, 4, 64, 8), (3, 64, 16, 1)):
        rows = tokens * hq // hkv
        block = 8 if rows <= 8 else 16 if rows <= 16 else 32
        assert lib.dscuda_flash_decode_workspace_bytes(batch, tokens, hq, hkv) == 888 * block * 129 * 4 + batch * hkv * -(-rows // block) * 8
    assert lib.dscuda_flash_cross_forward_workspace_bytes(2, 50, 70, 8, 2) == 0
    assert lib.dscuda_flash_cross_backward_workspace_bytes(2, 50, 70, 8, 2) == 2 * 50 * 8 * 8
