"""Entry points of the 8-bit paged cache and the paged chunk attention, as the C
ABI has them: argument blocks laid out as the header and the binding's packers say,
and what they refuse, with a message (CPU only: no kernel is launched)."""

import ctypes
import math
import os
import subprocess

import pytest

from helpers import REPO

BASE = 0x10000
E4M3, BF, H, F32 = 3, 1, 2, 0


@pytest.fixture(scope="module")
def bridge():
    from mac_attention.integrations.sglang import bridge as b

    if not os.path.exists(b.LIB_PATH):
        pytest.fail(f"{b.LIB_PATH} is not built; run __graft_entry__.build()")
    return b


@pytest.fixture(scope="module")
def lib(bridge):
    return bridge.load_library()


STRUCTS = [("MacPagedCache", "_pack_cache"), ("MacPagedRopeArgs", "_pack_rope"), ("MacPagedAttentionArgs", "_pack_attention")]


@pytest.mark.parametrize("name", [s[0] for s in STRUCTS])
def test_struct_layout_matches_header(bridge, tmp_path, name):
    cls = getattr(bridge, name)
    fields = [f[0] for f in cls._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "mac_attention_amd.h"', "int main(void) {",
           f'printf("size %zu\\n", sizeof({name}));']
    src += [f'printf("{f} %zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0; }"]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src))
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(c), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(out[f]) == getattr(cls, f).offset, f


@pytest.mark.parametrize("name,pack", STRUCTS)
def test_packed_blocks_equal_the_mirrors(bridge, name, pack):
    cls, pack = getattr(bridge, name), getattr(bridge, pack)
    floats = (ctypes.c_float, ctypes.c_double)
    values = [0.5 + i if t in floats else i + 3 for i, (_, t) in enumerate(cls._fields_)]
    mirror = cls.from_buffer_copy(pack(*values))
    assert [getattr(mirror, f) for f, _ in cls._fields_] == values
    with pytest.raises(RuntimeError, match="out of range"):
        pack(1 << 40, *values[1:])


def make_cache(bridge, **kw):
    c = bridge.MacPagedCache()
    c.struct_size, c.abi_version = ctypes.sizeof(c), bridge.ABI_VERSION
    c.k_cache, c.v_cache, c.kv_scales = BASE, BASE * 2, BASE * 3
    c.num_pages, c.page_size, c.Hkv, c.D, c.cache_dtype = 8, 16, 2, 128, E4M3
    c.k_page_stride, c.k_slot_stride, c.k_head_stride = 16 * 256, 256, 128
    c.v_page_stride, c.v_slot_stride, c.v_head_stride = 16 * 256, 256, 128
    c.k_scale = c.v_scale = 1.0
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def refused(lib, rc, text):
    message = lib.mac_last_error().decode()
    assert rc != 0 and text in message, (rc, text, message)


CACHE = [
    (dict(struct_size=8), "struct_size"), (dict(abi_version=1), "abi_version"), (dict(num_pages=0), "num_pages"),
    (dict(page_size=0), "power of two"), (dict(page_size=12), "power of two"), (dict(page_size=-16), "power of two"),
    (dict(kv_scales=BASE + 1), "2-byte"), (dict(k_scale=2.0), "takes no k_scale"),
    (dict(kv_scales=None, v_scale=0.0), "positive"), (dict(kv_scales=None, k_scale=-1.0), "positive"),
    (dict(kv_scales=None, k_scale=math.nan), "positive"), (dict(kv_scales=None, v_scale=math.inf), "positive"),
    (dict(k_cache=None), "null pointer"), (dict(v_cache=BASE + 8), "16-byte aligned"), (dict(k_slot_stride=264), "multiples of 16"),
]
CACHE8 = CACHE + [
    (dict(cache_dtype=BF, kv_scales=None), "e4m3"), (dict(Hkv=0), "positive"), (dict(D=40), "multiple of 16"),
    (dict(D=272), "multiple of 16"), (dict(D=0), "multiple of 16"), (dict(v_head_stride=-8), "multiples of 16"),
]


def write(lib, c, k=BASE * 4, v=BASE * 5, dtype=BF, locs=BASE * 6, tokens=1):
    return lib.mac_paged_cache_write_fp8(ctypes.byref(c) if c is not None else None, k, 256, 128, v, 256, 128, dtype, locs, 0, tokens, None)


def read(lib, c, locs=BASE * 4, rows=1, k=BASE * 5, v=BASE * 6, dtype=BF):
    return lib.mac_paged_cache_read_fp8(ctypes.byref(c) if c is not None else None, locs, 0, rows, k, v, dtype, None)


@pytest.mark.parametrize("change,text", CACHE8)
def test_writes_and_reads_refuse_bad_caches(bridge, lib, change, text):
    c = make_cache(bridge, **change)
    refused(lib, write(lib, c), text)
    refused(lib, read(lib, c), text)
    refused(lib, lib.mac_paged_rope_write_fp8(ctypes.byref(c), ctypes.byref(rope_args(bridge)), None), text)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(locs=None), "null pointer"), (dict(dtype=F32), "bfloat16 or float16"),
    (dict(dtype=E4M3), "bfloat16 or float16"), (dict(tokens=-1), ">= 0"), (dict(tokens=1 << 31), "too many rows"),
])
def test_writes_refuse(bridge, lib, change, text):
    refused(lib, write(lib, make_cache(bridge), **change), text)
    refused(lib, write(lib, None), "NULL")


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pointer"), (dict(locs=None), "null pointer"), (dict(dtype=E4M3), "dtype must be"), (dict(dtype=-1), "dtype must be"),
    (dict(rows=-1), ">= 0"), (dict(rows=1 << 31), "too many rows"), (dict(k=BASE + 8), "16-byte aligned"), (dict(v=BASE + 2), "16-byte aligned"),
])
def test_reads_refuse(bridge, lib, change, text):
    refused(lib, read(lib, make_cache(bridge), **change), text)
    refused(lib, read(lib, None), "NULL")


def test_nothing_to_do_is_no_error(bridge, lib):
    c = make_cache(bridge)
    assert write(lib, c, k=None, v=None, locs=None, tokens=0) == 0
    assert read(lib, c, locs=None, rows=0, k=None, v=None) == 0
    assert lib.mac_paged_rope_write_fp8(ctypes.byref(c), ctypes.byref(rope_args(bridge, tokens=0)), None) == 0
    for change in (dict(B=0), dict(total_q=0)):
        a = attention_args(bridge, q=None, out=None, **change)
        assert lib.mac_paged_chunk_attention_workspace(ctypes.byref(c), ctypes.byref(a)) == 0
        assert lib.mac_paged_chunk_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 0


def rope_args(bridge, **kw):
    a = bridge.MacPagedRopeArgs()
    a.struct_size, a.abi_version = ctypes.sizeof(a), bridge.ABI_VERSION
    a.q, a.k, a.v, a.q_out, a.cos_sin_cache, a.positions, a.cache_locs = (BASE * i for i in range(4, 11))
    a.q_stride0 = a.k_stride0 = a.v_stride0 = 1024
    a.q_stride1 = a.k_stride1 = a.v_stride1 = 128
    a.cos_sin_rows, a.cos_sin_stride0, a.tokens, a.Hq, a.rotary_dim, a.is_neox, a.dtype = 64, 128, 1, 8, 128, 1, BF
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(struct_size=4), "struct_size"), (dict(abi_version=9), "abi_version"), (dict(dtype=F32), "bfloat16 or float16"), (dict(Hq=0), "Hq"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=130), "rotary_dim"), (dict(cos_sin_rows=0), "empty"),
    (dict(q=None), "null pointer"), (dict(positions=None), "null pointer"), (dict(q_out=BASE + 8), "16-byte aligned"),
    (dict(tokens=-1), ">= 0"), (dict(tokens=1 << 31), "too many rows"), (dict(q_out=BASE * 4), "overlap"),
    (dict(q_out=BASE * 4 + 2032), "overlap"), (dict(q_out=BASE * 5 - 1008), "overlap"), (dict(q_out=BASE * 6 - 2032), "overlap"),
    (dict(q=BASE * 64, q_stride0=-1024, tokens=3, q_out=BASE * 64 - 4096), "overlap"),
])
def test_rope_writes_refuse(bridge, lib, change, text):
    c = make_cache(bridge)
    refused(lib, lib.mac_paged_rope_write_fp8(ctypes.byref(c), ctypes.byref(rope_args(bridge, **change)), None), text)
    refused(lib, lib.mac_paged_rope_write_fp8(ctypes.byref(c), None, None), "NULL")
    refused(lib, lib.mac_paged_rope_write_fp8(None, ctypes.byref(rope_args(bridge)), None), "NULL")


def attention_args(bridge, **kw):
    a = bridge.MacPagedAttentionArgs()
    a.struct_size, a.abi_version = ctypes.sizeof(a), bridge.ABI_VERSION
    a.q, a.qo_indptr, a.kv_lens, a.page_table, a.out, a.out_lse = (BASE * i for i in range(4, 10))
    a.q_stride0, a.q_stride1, a.table_stride = 1024, 128, 4
    a.total_q, a.B, a.Hq, a.table_rows, a.table_cols, a.q_dtype, a.window_left = 1, 1, 8, 1, 4, BF, -1
    a.sm_scale = 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attend(lib, c, a, workspace=BASE * 32, size=1 << 40):
    return lib.mac_paged_chunk_attention(ctypes.byref(c) if c is not None else None, ctypes.byref(a) if a is not None else None, workspace,
                                         size, None)


@pytest.mark.parametrize("change,text", CACHE + [
    (dict(cache_dtype=H, kv_scales=None), "q's type"), (dict(cache_dtype=BF), "belong to an e4m3"), (dict(D=96), "head_dim"), (dict(D=16), "head_dim"),
    (dict(Hkv=0), "multiple of Hkv"), (dict(Hkv=3), "multiple of Hkv"), (dict(num_pages=1 << 31), "31 bits"), (dict(v_head_stride=256), "same strides"),
    (dict(k_page_stride=1 << 32, v_page_stride=1 << 32), "2^32"), (dict(k_page_stride=-4096, v_page_stride=-4096), "2^32"),
    (dict(page_size=1 << 28), "2^30 keys"),
])
def test_attention_refuses_bad_caches(bridge, lib, change, text):
    refused(lib, attend(lib, make_cache(bridge, **change), attention_args(bridge)), text)


@pytest.mark.parametrize("change,text", [
    (dict(struct_size=4), "struct_size"), (dict(abi_version=9), "abi_version"), (dict(q_dtype=F32), "bfloat16 or float16"),
    (dict(Hq=0), "multiple of Hkv"), (dict(Hq=7), "multiple of Hkv"), (dict(B=-1), "B must be"), (dict(B=4097), "B must be"),
    (dict(total_q=-1), "total_q"), (dict(total_q=1 << 29), "total_q"), (dict(table_cols=-1), "2^30 keys"), (dict(table_rows=-1), "2^30 keys"),
    (dict(table_cols=1 << 26), "2^30 keys"), (dict(sm_scale=0.0), "sm_scale"), (dict(sm_scale=math.nan), "sm_scale"),
    (dict(sm_scale=1e300), "fit fp32"), (dict(logit_cap=-1.0), "logit_cap"), (dict(logit_cap=math.inf), "logit_cap"),
    (dict(logit_cap=1e60), "fit fp32"), (dict(logit_cap=1e-60), "fit fp32"), (dict(q=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(out_lse=None), "null pointer"), (dict(page_table=None), "null pointer"), (dict(q=BASE + 8), "16-byte aligned"),
    (dict(q_stride0=1020), "16-byte aligned"), (dict(out=BASE + 4), "16-byte aligned"),
    (dict(total_q=1 << 24, Hq=2), "total_q"), (dict(total_q=(1 << 24) - 1, Hq=64, B=4096), "too large"),
])
def test_attention_refuses(bridge, lib, change, text):
    c = make_cache(bridge)
    refused(lib, attend(lib, c, attention_args(bridge, **change)), text)
    refused(lib, attend(lib, None, attention_args(bridge)), "NULL")
    refused(lib, attend(lib, c, None), "NULL")


def test_attention_refuses_more_rows_and_heads_than_a_launch_has_workgroups(bridge, lib):
    c = make_cache(bridge, Hkv=2048)
    refused(lib, attend(lib, c, attention_args(bridge, Hq=2048, total_q=512 * 16, B=512)), "batch too large")


def test_attention_refuses_small_workspaces(bridge, lib):
    c, a = make_cache(bridge), attention_args(bridge)
    need = lib.mac_paged_chunk_attention_workspace(ctypes.byref(c), ctypes.byref(a))
    assert need > 0
    refused(lib, attend(lib, c, a, size=need - 1), "workspace too small")
    refused(lib, attend(lib, c, a, workspace=BASE + 8), "misaligned")
    refused(lib, attend(lib, c, a, workspace=None, size=need), "workspace too small")
    assert lib.mac_paged_chunk_attention_workspace(ctypes.byref(make_cache(bridge, D=32)), ctypes.byref(a)) == -1


def test_binding_refuses_host_tensors(bridge):
    torch = pytest.importorskip("torch")
    ext = bridge.load_mac_paged_cache_extension(False)
    f8 = torch.zeros(4, 8, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    rows, locs = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3, dtype=torch.int32)
    scales = torch.zeros(4, 2, 8, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ext.mac_paged_cache_write_fp8(rows, rows, f8, f8, scales, locs)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ext.mac_paged_cache_read_fp8(f8, f8, scales, locs)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ext.mac_paged_rope_write_fp8(rows, rows, rows, f8, f8, scales, torch.zeros(8, 64), locs, locs)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ext.mac_paged_chunk_attention(rows, f8, f8, locs, locs[:2], torch.zeros(2, 1, dtype=torch.int32), 1.0, kv_scales=scales)
