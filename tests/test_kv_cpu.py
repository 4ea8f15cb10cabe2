"""What the paged key/value cache refuses before anything is launched, and its host-side helpers (no GPU needed)."""
import ctypes
import math

import numpy as np
import pytest

from mlxl3_b200 import _lib, kv
from oracle import kv as okv

BASE = 1 << 20                                       # stands for a device address; nothing may look behind it
F16, BF16, F32 = 9, 12, 10


def cache(**change):
    args = dict(pages=4, page_size=16, kv_heads=2, head_dim=128, dtype=F16, bits=16, d_k=BASE, d_v=BASE, d_k_scale=BASE, d_v_scale=BASE)
    args.update(change)
    return kv.KvCache(**args)


def batch(**change):
    args = dict(d_row_start=BASE, d_length=BASE, d_page_table=BASE, batch=2, table_width=4, rows=3)
    args.update(change)
    return kv.KvBatch(**args)


class Workspace:
    def __init__(self, ptr=BASE, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


def append(c=None, b=None, rope=None, **change):
    args = dict(d_k=BASE, d_v=BASE, d_q=BASE, heads=4, d_q_out=BASE)
    args.update(change)
    kv.append(c or cache(), b or batch(), rope=rope, **args)


def attention(c=None, b=None, workspace=None, **change):
    args = dict(d_q=BASE, heads=4, scale=0.1, d_out=BASE)
    args.update(change)
    kv.attention(c or cache(), b or batch(), workspace=workspace or Workspace(), **args)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=F32), "f16 or bf16"), (dict(bits=5), "16, 8 or 4 bits"), (dict(head_dim=96), "head dimension of 64 or 128"),
    (dict(pages=0), "invalid paged cache"), (dict(page_size=0), "invalid paged cache"), (dict(kv_heads=-1), "invalid paged cache"),
    (dict(d_v=0), "NULL buffer"), (dict(bits=8, d_k_scale=0), "NULL buffer"), (dict(d_k=BASE + 8), "16-byte aligned"),
    (dict(bits=4, d_v_scale=BASE + 2), "4-byte aligned")])
def test_caches_that_are_refused(change, message):
    for call in (append, attention, lambda c: kv.read(c, batch(), F32, BASE, BASE)):
        with pytest.raises(_lib.B200Exl3Error, match=message):
            call(cache(**change))


@pytest.mark.parametrize("change,message", [
    (dict(batch=0), "invalid batch"), (dict(rows=0), "invalid batch"), (dict(rows=1 << 31), "invalid batch"), (dict(table_width=0), "invalid batch"),
    (dict(table_width=(1 << 26) + 1), "2\\^30 tokens"), (dict(d_length=0), "NULL buffer"), (dict(d_page_table=BASE + 2), "4-byte aligned")])
def test_batches_that_are_refused(change, message):
    for call in (append, attention, lambda b: kv.read(cache(), b, F32, BASE, BASE)):
        with pytest.raises(_lib.B200Exl3Error, match=message):
            call(b=batch(**change)) if call in (append, attention) else call(batch(**change))


@pytest.mark.parametrize("change,message", [
    (dict(heads=-1), "head counts"), (dict(d_q=0), "NULL buffer"), (dict(d_v=0), "NULL buffer"), (dict(d_k=BASE + 2), "16-byte aligned"),
    (dict(q_stride=504), "cannot lie"), (dict(k_stride=260), "cannot lie"), (dict(v_stride=-256), "cannot lie"), (dict(q_stride=520), "one stride"),
    (dict(rope=kv.Rope(BASE, 24)), "multiple of 16"), (dict(rope=kv.Rope(BASE, 144)), "multiple of 16"), (dict(rope=kv.Rope(0, 128)), "NULL buffer"),
    (dict(rope=kv.Rope(BASE + 4, 128)), "8-byte aligned"), (dict(rope=kv.Rope(BASE, 128, False, math.inf)), "magnitude")])
def test_appends_that_are_refused(change, message):
    with pytest.raises(_lib.B200Exl3Error, match=message):
        append(**change)


@pytest.mark.parametrize("args,message", [((7, BASE, BASE), "unsupported dtype"), ((F16, 0, 0), "NULL buffer"), ((F16, BASE + 4, 0), "16-byte aligned")])
def test_reads_that_are_refused(args, message):
    with pytest.raises(_lib.B200Exl3Error, match=message):
        kv.read(cache(), batch(), *args)


@pytest.mark.parametrize("change,message", [
    (dict(heads=3), "head counts"), (dict(heads=0), "head counts"), (dict(scale=math.nan), "scale"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(window=-1), "window"), (dict(max_new=-1), "new tokens"),
    (dict(d_out=0), "NULL buffer"), (dict(out_stride=8), "cannot lie"), (dict(d_q=BASE + 2), "16-byte aligned"),
    (dict(workspace=Workspace(nbytes=1 << 14)), "workspace too small"), (dict(workspace=Workspace(ptr=0)), "workspace too small"),
    (dict(workspace=Workspace(ptr=BASE + 8)), "16-byte aligned")])
def test_attention_that_is_refused(change, message):
    with pytest.raises(_lib.B200Exl3Error, match=message):
        attention(**change)


def test_missing_arguments_are_refused():
    lib = _lib.load()
    c, b = cache(), batch()
    out = ctypes.c_size_t()
    assert lib.b200exl3_kv_append(None, ctypes.byref(b), None, BASE, 0, 4, BASE, 0, BASE, 0, BASE, 0, None) == -1
    assert lib.b200exl3_kv_append(ctypes.byref(c), None, None, BASE, 0, 4, BASE, 0, BASE, 0, BASE, 0, None) == -1
    assert lib.b200exl3_kv_read(ctypes.byref(c), None, F32, BASE, BASE, None) == -1
    assert lib.b200exl3_kv_attention(ctypes.byref(c), None, BASE, 0, 4, 0.1, 0, 0, BASE, 0, BASE, 1 << 40, None) == -1
    assert lib.b200exl3_kv_attention_workspace_bytes(ctypes.byref(c), 4, 1, None) == -1
    assert lib.b200exl3_kv_attention_workspace_bytes(None, 4, 1, ctypes.byref(out)) == -1
    with pytest.raises(_lib.B200Exl3Error, match="head counts"):
        kv.attention_workspace_bytes(c, 5, 1)


def test_workspace_covers_smaller_calls():
    for bits in (16, 8, 4):
        for d in (64, 128):
            c = cache(bits=bits, head_dim=d)
            sizes = [kv.attention_workspace_bytes(c, 16, n) for n in (1, 2, 3, 16, 17, 100, 5000)]
            assert sizes == sorted(sizes)


def test_rope_turns():
    turns = kv.rope_turns(64, 10000.0)
    assert turns.dtype == np.float64 and turns.shape == (32,)
    assert abs(turns[0] * 2 * math.pi - 1.0) < 1e-15 and abs(turns[16] * 2 * math.pi - 0.01) < 1e-15
    assert np.array_equal(kv.rope_turns(64, 10000.0, 8.0), turns / 8.0)
    part = kv.rope_turns(64, 10000.0, 8.0, 1.0, 4.0, 2048)
    fast, slow = turns * 2048 > 4.0, turns * 2048 < 1.0
    assert np.array_equal(part[fast], turns[fast]) and np.array_equal(part[slow], turns[slow] / 8.0)
    between = ~fast & ~slow
    assert between.any() and (part[between] < turns[between]).all() and (part[between] > turns[between] / 8.0).all()
    for bad in ((63, 1e4), (64, 1.0), (0, 1e4), (64, 1e4, 0.0), (64, 1e4, 8.0, 4.0, 1.0, 2048)):
        with pytest.raises(_lib.B200Exl3Error):
            kv.rope_turns(*bad)


def test_oracle_rotates_and_packs():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 64))
    turns = kv.rope_turns(32, 10000.0)
    for interleaved in (False, True):
        y = okv.rope(x, 1000003, turns, interleaved)
        assert np.array_equal(y[:, 32:], x[:, 32:]) and np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-13)
        a, b = okv.rope(x, 17, turns, interleaved), okv.rope(x[::-1], 5, turns, interleaved)
        a2, b2 = okv.rope(x, 112, turns, interleaved), okv.rope(x[::-1], 100, turns, interleaved)
        assert np.allclose((a * b).sum(-1), (a2 * b2).sum(-1), rtol=1e-12)      # only the distance counts
    for bits in (8, 4):
        codes, scale = okv.quantise(x, bits)
        assert np.array_equal(okv.unpack(okv.pack(codes, bits), bits), codes)
        assert (np.abs(codes * scale[:, None].astype(np.float64) - x) <= scale[:, None] * 0.5001).all()


@pytest.mark.parametrize("mirror,struct_name", [(kv.KvCache, "b200exl3_kv_cache"), (kv.KvBatch, "b200exl3_kv_batch"), (kv.Rope, "b200exl3_rope")])
def test_ctypes_mirror_matches_the_header(mirror, struct_name):
    from tests.test_struct_layout import c_layout
    layout, total = c_layout(struct_name)
    assert [(name, getattr(mirror, name).offset, getattr(mirror, name).size) for name, _ in mirror._fields_] == layout
    assert ctypes.sizeof(mirror) == total
