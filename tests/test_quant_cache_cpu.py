"""CPU tests of the quantised-cache entry points: the ctypes mirrors have the C layout, and arguments that the
header rules out come back as status codes before anything touches a GPU."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

import quant_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20  # an aligned address that nobody follows


def test_ctypes_structs_match_c_layout(native_lib):
    mirrors = {"da_kv_rows_args_t": native_lib.KvRowsArgs, "da_quant_decode_args_t": native_lib.QuantDecodeArgs,
               "da_prefix_decode_args_t": native_lib.PrefixDecodeArgs}
    body = "".join('printf("%%zu\\n", sizeof(%s));' % t + "".join('printf("%%zu\\n", offsetof(%s, %s));' % (t, f[0]) for f in m._fields_)
                   for t, m in mirrors.items())
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write('#include <stdio.h>\n#include <stddef.h>\n#include "decoding_attn_b200.h"\nint main(){%s return 0;}' % body)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = list(map(int, subprocess.check_output([exe]).split()))
    want = []
    for m in mirrors.values():
        want += [ctypes.sizeof(m)] + [getattr(m, f[0]).offset for f in m._fields_]
    assert got == want


def rows_args(native_lib, **change):
    a = native_lib.KvRowsArgs(struct_size=ctypes.sizeof(native_lib.KvRowsArgs), kv_dtype=2, x_dtype=1, k=PTR, v=PTR, k_cache=PTR,
                              v_cache=PTR, k_scale=PTR, v_scale=PTR, slots=PTR, tokens=4, cache_rows=8, head_k=2, dim=128)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [
    {"struct_size": 8}, {"kv_dtype": 0}, {"kv_dtype": 4}, {"x_dtype": -1}, {"x_dtype": 3}, {"k": None}, {"v_cache": None},
    {"v_scale": None}, {"tokens": -1}, {"cache_rows": -1}, {"head_k": 0}, {"tokens": 1 << 31}, {"slots": None, "tokens": 9},
    {"k": PTR + 8}, {"v_cache": PTR + 4}, {"k_scale": PTR + 2}, {"slots": PTR + 4}, {"k_row_stride": 128}, {"v_row_stride": 260},
    {"head_k": 1 << 31, "tokens": 1}])
def test_row_arguments_are_refused(native_lib, change):
    lib = native_lib.lib()
    for call in (lib.da_kv_cache_write, lib.da_kv_cache_read):
        assert call(ctypes.byref(rows_args(native_lib, **change))) == native_lib.DA_ERR_INVALID_ARG
        assert lib.da_last_error()


def test_row_arguments_by_direction_and_dim(native_lib):
    lib = native_lib.lib()
    assert lib.da_kv_cache_write(ctypes.byref(rows_args(native_lib, x_dtype=2))) == native_lib.DA_ERR_INVALID_ARG
    assert lib.da_kv_cache_write(None) == native_lib.DA_ERR_INVALID_ARG
    for dim in (0, 32, 80, 112, 512, 576):
        assert lib.da_kv_cache_read(ctypes.byref(rows_args(native_lib, dim=dim))) == native_lib.DA_ERR_UNSUPPORTED
    # no tokens: nothing to do, nothing launched
    before = native_lib.launch_count()
    for call in (lib.da_kv_cache_write, lib.da_kv_cache_read):
        assert call(ctypes.byref(rows_args(native_lib, tokens=0, k=None, v=None, slots=None))) == native_lib.DA_OK
    assert native_lib.launch_count() == before


def quant_args(native_lib, **change):
    a = native_lib.QuantDecodeArgs(struct_size=ctypes.sizeof(native_lib.QuantDecodeArgs), is_bf16=1, kv_dtype=1, q=PTR, k=PTR, v=PTR,
                                   k_scale=PTR, v_scale=PTR, o=PTR, cu_seq_k=PTR, rows=100, batch=2, head_q=8, head_k=2, dim=128,
                                   workspace=PTR, workspace_bytes=1 << 30)
    for name, value in change.items():
        setattr(a, name, value)
    return a


PAGED = {"block_table": PTR, "block_table_stride": 4, "table_blocks": 4, "page_size": 16}


@pytest.mark.parametrize("change", [
    {"struct_size": 0}, {"kv_dtype": 0}, {"kv_dtype": 9}, {"batch": 0}, {"batch": 65536}, {"head_q": 7}, {"head_k": 0},
    {"head_q": 1 << 17, "head_k": 1}, {"rows": -1}, {"rows": 1 << 31}, {"q": None}, {"o": None}, {"cu_seq_k": None}, {"k": None},
    {"v_scale": None}, {"q": PTR + 8}, {"o": PTR + 2}, {"workspace": PTR + 4}, {"lse": PTR + 1}, {"q_row_stride": 100},
    {"o_row_stride": 1028}, {"page_size": 16}, {"table_blocks": 3}, {**PAGED, "table_blocks": 0}, {**PAGED, "table_blocks": 5}])
def test_decode_arguments_are_refused(native_lib, change):
    lib = native_lib.lib()
    assert lib.da_quant_decode_fwd(ctypes.byref(quant_args(native_lib, **change))) == native_lib.DA_ERR_INVALID_ARG
    assert lib.da_quant_decode_workspace_bytes(ctypes.byref(quant_args(native_lib, **change))) == 0


def test_decode_shapes_are_refused(native_lib):
    lib = native_lib.lib()
    for change in ({"dim": 80}, {"dim": 576}, {**PAGED, "page_size": 0}, {**PAGED, "page_size": 24}):
        assert lib.da_quant_decode_fwd(ctypes.byref(quant_args(native_lib, **change))) == native_lib.DA_ERR_UNSUPPORTED
    assert lib.da_quant_decode_fwd(None) == native_lib.DA_ERR_INVALID_ARG


def prefix_args(native_lib, **change):
    a = native_lib.PrefixDecodeArgs(struct_size=ctypes.sizeof(native_lib.PrefixDecodeArgs), is_bf16=1, q=PTR, k_prefix=PTR, v_prefix=PTR,
                                    k=PTR, v=PTR, o=PTR, cu_seq_k=PTR, prefix_len=50, prefix_rows=64, rows=100, batch=2, head_q=8,
                                    head_k=2, dim=128, workspace=PTR, workspace_bytes=1 << 30)
    for name, value in change.items():
        setattr(a, name, value)
    return a


SCALES = {"kv_dtype": 2, "k_scale": PTR, "v_scale": PTR}


@pytest.mark.parametrize("change", [
    {"struct_size": 0}, {"kv_dtype": -1}, {"kv_dtype": 4}, {"kv_dtype": 2}, {"k_scale": PTR}, {**SCALES, "v_scale": None},
    {"batch": 0}, {"batch": 65536}, {"head_q": 7}, {"head_k": 0}, {"prefix_len": -1}, {"prefix_len": (1 << 30) + 1},
    {"prefix_len": 65}, {"rows": 1 << 31}, {"prefix_rows": 1 << 31}, {"q": None}, {"o": None}, {"cu_seq_k": None},
    {"k_prefix": None}, {"v": None}, {"v_prefix": PTR + 8}, {"workspace": PTR + 4}, {"cu_seq_k": PTR + 2}, {"q_row_stride": 1028},
    {"k_prefix_row_stride": 128}, {"v_row_stride": 260}, {**SCALES, "k_row_stride": 512}, {"prefix_page_size": 16},
    {"page_size": 16}, {**PAGED, "table_blocks": 0}, {**PAGED, "block_table_stride": 3}])
def test_prefix_arguments_are_refused(native_lib, change):
    lib = native_lib.lib()
    assert lib.da_prefix_decode_fwd(ctypes.byref(prefix_args(native_lib, **change))) == native_lib.DA_ERR_INVALID_ARG
    assert lib.da_prefix_decode_workspace_bytes(ctypes.byref(prefix_args(native_lib, **change))) == 0


def test_prefix_shapes_are_refused(native_lib):
    lib = native_lib.lib()
    for change in ({"dim": 256}, {"dim": 80}, {"head_q": 258}, {"prefix_table": PTR}, {"prefix_table": PTR, "prefix_page_size": 8},
                   {"prefix_table": PTR, "prefix_page_size": 48}, {**PAGED, "page_size": 12},
                   {"batch": 65535, "head_q": 128, "prefix_table": PTR, "prefix_page_size": 64, "prefix_len": 1 << 30}):
        assert lib.da_prefix_decode_fwd(ctypes.byref(prefix_args(native_lib, **change))) == native_lib.DA_ERR_UNSUPPORTED
    assert lib.da_prefix_decode_fwd(None) == native_lib.DA_ERR_INVALID_ARG


@pytest.mark.parametrize("kind", ["fp8", "int8", "int4"])
def test_plain_form_of_the_tests(kind):
    """The tests' own quantiser: codes stay in range, no element is further off than half a step of its code."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, 3, 64, generator=g).to(torch.bfloat16)
    codes, scale = ref.quantise(x, kind)
    assert codes.abs().max() <= ref.QMAX[kind]
    assert torch.equal(ref.unpack(ref.pack(codes, kind), kind), codes)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(codes.abs().clamp(min=2.0 ** -9))), min=-6) - 3) if kind == "fp8" else torch.ones_like(codes)
    off = (x.double() / scale.double().unsqueeze(-1) - codes).abs()
    # (scale and its inverse are rounded apart: two half steps of fp32; the codes above a power of two sit on its finer side)
    assert (off <= step / 2 * (1 + 2.0 ** -10) + codes.abs() * 2.0 ** -22).all()
