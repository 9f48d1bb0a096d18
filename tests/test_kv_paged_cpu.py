"""The paged cache's host side (include/kv_paged.h): declared symbols, shape
checks, and every refusal of a call, on a handle without a device, so nothing
here launches a kernel."""
import ctypes
import os
import re

import pytest

import pk_b200
from conftest import ROOT


def handle(**kw):
    a = dict(n_heads=8, n_kv_heads=2, head_size=64, qtype=pk_b200.F16, page_tokens=16, n_pages=10, max_requests=4,
             max_blocks=5, device=-1)
    a.update(kw)
    return pk_b200.KvPaged(**a)


def test_declared_symbols_are_exported():
    src = open(os.path.join(ROOT, "include", "kv_paged.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = set(re.findall(r"\b(kv_paged_[a-z_]+)\s*\(", src))
    assert names == set(pk_b200.KV_PAGED_EXPORTS)
    for n in names:
        assert hasattr(pk_b200.lib(), n)


def test_shape_layout(tmp_path):
    import subprocess
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include "kv_paged.h"\nint main(void){printf("%zu %zu %zu\\n",'
                   'sizeof(KvPagedShape),offsetof(KvPagedShape,type),offsetof(KvPagedShape,page_stride));}\n')
    exe = tmp_path / "p"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(pk_b200.KvPagedShape), pk_b200.KvPagedShape.type.offset,
                                     pk_b200.KvPagedShape.page_stride.offset]


@pytest.mark.parametrize("change,why", [
    (dict(qtype=pk_b200.Q8_0), "type must be"),
    (dict(n_heads=7), "multiple of the key-value heads"),
    (dict(n_heads=0), "multiple of the key-value heads"),
    (dict(n_kv_heads=0), "multiple of the key-value heads"),
    (dict(head_size=60), "head size"),
    (dict(head_size=264), "head size"),
    (dict(head_size=0), "head size"),
    (dict(page_tokens=0), "Pages and page size"),
    (dict(n_pages=0), "Pages and page size"),
    (dict(n_pages=1 << 28, page_tokens=8), "Pages and page size"),
    (dict(max_requests=0), "block table"),
    (dict(max_requests=4097), "block table"),
    (dict(max_blocks=0), "blocks"),
    (dict(max_blocks=1 << 28, page_tokens=8, n_pages=1), "blocks"),
    (dict(strides=(16 * 128, 128, 60)), "multiples of 16 bytes"),
    (dict(strides=(16 * 128, 120, 64)), "overlap"),
    (dict(strides=(16 * 128 - 8, 128, 64)), "overlap"),
    (dict(strides=(16 * 128, 128, 0)), "overlap"),
    (dict(strides=(1 << 33, 128, 64)), "64 GB"),
    (dict(device=-2), "Invalid device"),
])
def test_shapes_refused(change, why):
    with pytest.raises(RuntimeError, match=why):
        handle(**change)


@pytest.mark.parametrize("strides", [(0, 0, 0), (16 * 128, 128, 64), (16 * 128, 64, 16 * 64), (128, 128 * 10, 64),
                                     (4096, 136, 64), (1 << 31, 128, 64)])
def test_shapes_taken(strides):
    handle(strides=strides).close()


P = 1 << 20  # a pointer on 16 bytes that nothing reads


def call(kv, name, **change):
    a = dict(
        map=dict(len_ptr=P, start=P, end=P, n=4, table=P, free_pages=P, n_free=P, n_free_out=P, max_rows=9, row_request=P,
                 row_pos=P, row_slot=P, row0=P),
        append=dict(q=P, k=P, v=P, row_pos=P, row_slot=P, n=3, q_out=P, k_pool=P, v_pool=P, rope_cs=P, rope_dim=64,
                    rope_len=10),
        attend=dict(q=P, k_pool=P, v_pool=P, table=P, n_requests=4, row_request=P, row_pos=P, n=3, scale=0.1,
                    out=2 * P),
    )[name]
    a.update(change)
    with pytest.raises(RuntimeError) as e:
        getattr(kv, name)(**a)
    return str(e.value)


@pytest.mark.parametrize("name,change,why", [
    *[("map", {k: 0}, "NULL") for k in ("len_ptr", "start", "end", "table", "free_pages", "n_free", "n_free_out", "row0")],
    ("map", dict(n=0), "requests"), ("map", dict(n=5), "requests"), ("map", dict(max_rows=-1), "room"),
    ("map", dict(row_slot=0), "room"),
    *[("append", {k: 0}, "NULL") for k in ("q", "k", "v", "row_pos", "row_slot", "q_out", "k_pool", "v_pool")],
    ("append", dict(n=-1), "negative"), ("append", dict(rope_dim=63), "rotary"), ("append", dict(rope_dim=66), "rotary"),
    ("append", dict(rope_dim=-2), "rotary"), ("append", dict(rope_cs=0), "rotary"), ("append", dict(rope_len=0), "rotary"),
    ("append", dict(q_stride=508), "stride"), ("append", dict(kv_stride=124), "stride"),
    ("append", dict(q_stride=514), "stride"), ("append", dict(kv_stride=129), "stride"),
    *[("append", {k: P + 4}, "16 bytes") for k in ("q", "k", "v", "q_out", "k_pool", "v_pool", "rope_cs")],
    *[("attend", {k: 0}, "NULL") for k in ("q", "k_pool", "v_pool", "table", "row_request", "row_pos", "out")],
    ("attend", dict(n=-1), "rows"), ("attend", dict(n=65536), "rows"), ("attend", dict(n_requests=0), "requests"),
    ("attend", dict(n_requests=5), "requests"), ("attend", dict(scale=float("nan")), "scale"),
    ("attend", dict(scale=float("inf")), "scale"), ("attend", dict(q_stride=500), "stride"),
    ("attend", dict(q_stride=514), "stride"), ("attend", dict(out=P), "overlaps"),
    ("attend", dict(out=P + 512 * 4 * 3 - 16), "overlaps"),
    *[("attend", {k: P + 8}, "16 bytes") for k in ("q", "k_pool", "v_pool", "out")],
    *[("map", {k: P + 2}, "4 bytes") for k in ("len_ptr", "start", "end", "table", "free_pages", "n_free", "n_free_out",
                                               "row_request", "row_pos", "row_slot", "row0")],
    *[("append", {k: P + 2}, "4 bytes") for k in ("row_pos", "row_slot")],
    *[("attend", {k: P + 2}, "4 bytes") for k in ("table", "row_request", "row_pos")],
    *[("append", dict(q_out=P + d), "overlaps") for d in (16, 2048, 3 * 2048 - 16, -16, 16 - 3 * 2048)],
    ("append", dict(q_stride=1024, q_out=P + 2 * 4096 + 2048 - 16), "overlaps"),
])
def test_calls_refused(name, change, why):
    kv = handle()
    assert why in call(kv, name, **change)
    assert why in kv.last_error()
    kv.close()


def test_good_calls_reach_the_device_check():
    kv = handle()
    assert "no device" in call(kv, "map")
    assert "no device" in call(kv, "map", max_rows=0, row_request=0, row_pos=0, row_slot=0)
    assert "no device" in call(kv, "append")
    assert "no device" in call(kv, "append", q=0, q_out=0, rope_cs=0, rope_dim=0, rope_len=0)
    assert "no device" in call(kv, "append", q_stride=768, kv_stride=768)
    for d in (3 * 2048, -3 * 2048):
        assert "no device" in call(kv, "append", q_out=P + d)
    assert "no device" in call(kv, "attend")
    assert "no device" in call(kv, "attend", out=P + 512 * 4 * 3)
    assert kv.error() == -1
    kv.close()


def test_null_handle():
    L = pk_b200.lib()
    L.kv_paged_close(None)
    assert L.kv_paged_last_error(None) == b"" and L.kv_paged_error(None) == -1
    assert L.kv_paged_open(None, 0, None, 0) is None
    assert L.kv_paged_map(None, *[None] * 3, 1, *[None] * 4, 0, *[None] * 5) == 0
    assert L.kv_paged_attend(None, *[None] * 4, 1, None, None, 1, 1.0, None, 0, None) == 0
    assert L.kv_paged_append(None, *[None] * 5, 1, *[None] * 4, 0, 0, 0, 0, None) == 0


def test_no_device_fails_cleanly():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    with pytest.raises(RuntimeError, match="CUDA"):
        handle(device=0)


def test_engine_paged_calls_without_a_model():
    L = pk_b200.lib()
    err = ctypes.create_string_buffer(64)
    assert L.engine_batch_open_paged(None, 4, 16, 8, err, 64) == 0 and err.value == b"No model."
    assert L.engine_batch_release(None, 0) == 0
    assert L.engine_batch_free_pages(None) == -1
