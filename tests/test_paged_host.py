"""The paged operators' host side, no device: frequency tables against their formulas, and every refusal by name."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from itak_torch_rebuild_b200 import CudaComputeError, _lib, paged

BASE = 500000.0


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.load()


@pytest.mark.parametrize("rot", [2, 64, 128, 256])
def test_plain_linear_and_base_tables(lib, rot):
    i = np.arange(rot // 2, dtype=np.float64)
    plain = BASE ** (-2 * i / rot)
    f, m = paged.rope_table(rot, BASE)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert m == 1.0
    f, m = paged.rope_table(rot, BASE, scaling="linear", factor=4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-14)
    assert m == 1.0
    if rot > 2:
        f, _ = paged.rope_table(rot, BASE, scaling="base", factor=4.0)
        assert f[0] == 1.0
        np.testing.assert_allclose(f[-1], plain[-1] / 4, rtol=1e-12)  # the slowest pair: as interpolated
        np.testing.assert_allclose(f, (BASE * 4.0 ** (rot / (rot - 2))) ** (-2 * i / rot), rtol=1e-12)


def test_banded_table(lib):
    rot, ctx, factor, low, high = 128, 8192.0, 8.0, 1.0, 4.0
    i = np.arange(64, dtype=np.float64)
    plain = BASE ** (-2 * i / rot)
    f, m = paged.rope_table(rot, BASE, scaling="bands", factor=factor, original_context=ctx, low=low, high=high)
    wave = 2 * math.pi / plain
    for j in range(64):
        if wave[j] < ctx / high:
            want = plain[j]
        elif wave[j] > ctx / low:
            want = plain[j] / factor
        else:
            s = (ctx / wave[j] - low) / (high - low)
            want = (1 - s) * plain[j] / factor + s * plain[j]
        assert f[j] == pytest.approx(want, rel=1e-13)
    assert m == 1.0 and (f[1:] <= f[:-1]).all()


def test_ramp_table_and_magnitude(lib):
    rot, ctx, factor, low, high = 128, 4096.0, 16.0, 1.0, 32.0
    f, m = paged.rope_table(rot, 10000.0, scaling="ramp", factor=factor, original_context=ctx, low=low, high=high)
    plain = 10000.0 ** (-2 * np.arange(64) / rot)
    a = math.floor(rot * math.log(ctx / (high * 2 * math.pi)) / (2 * math.log(10000.0)))
    b = math.ceil(rot * math.log(ctx / (low * 2 * math.pi)) / (2 * math.log(10000.0)))
    for j in range(64):
        gone = min(1.0, max(0.0, (j - a) / (b - a)))
        assert f[j] == pytest.approx(plain[j] * (1 - gone) + plain[j] / factor * gone, rel=1e-13)
    assert m == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-7)
    assert paged.rope_table(rot, 10000.0, scaling="ramp", factor=factor, original_context=ctx, low=low, high=high, magnitude=1.5)[1] == 1.5


@pytest.mark.parametrize("rot,base,ctx,behind", [(128, 10000.0, 65536.0, True), (128, 10000.0, 131072.0, True), (64, 10000.0, 65536.0, True),
                                                 (64, 10000.0, 1e9, True), (128, 10000.0, 32768.0, False), (4, 500000.0, 8192.0, True),
                                                 (2, 500000.0, 8192.0, True), (128, 500000.0, 8192.0, False)])
def test_ramp_whose_upper_pair_lies_behind_the_last(lib, rot, base, ctx, behind):
    """Slow pairs that make more than `low` turns over the original context: the ramp's upper end is not moved to the last
    pair, only to rotary_dim - 1."""
    factor, low, high = 8.0, 1.0, 32.0
    f, _ = paged.rope_table(rot, base, scaling="ramp", factor=factor, original_context=ctx, low=low, high=high)
    a = max(0.0, math.floor(rot * math.log(ctx / (high * 2 * math.pi)) / (2 * math.log(base))))
    b = min(rot - 1.0, math.ceil(rot * math.log(ctx / (low * 2 * math.pi)) / (2 * math.log(base))))
    assert (b > rot / 2 - 1) == behind
    for j in range(rot // 2):
        plain = base ** (-2 * j / rot)
        gone = min(1.0, max(0.0, (j - a) / max(b - a, 1e-3)))
        assert f[j] == pytest.approx(plain * (1 - gone) + plain / factor * gone, rel=1e-13), j
    if behind:
        assert f[-1] > base ** (2.0 / rot - 1.0) / factor * 1.0000001


def test_pair_factors(lib):
    pf = np.linspace(1, 9, 32)
    f, _ = paged.rope_table(64, BASE, scaling="pairs", pair_factors=pf)
    np.testing.assert_allclose(f, BASE ** (-2 * np.arange(32) / 64) / pf.astype(np.float32), rtol=1e-13)


def test_factor_one_changes_nothing(lib):
    plain, _ = paged.rope_table(128, BASE)
    for kind in ("linear", "base", "bands", "ramp"):
        f, m = paged.rope_table(128, BASE, scaling=kind, factor=1.0, original_context=8192.0, low=1.0, high=4.0)
        np.testing.assert_allclose(f, plain, rtol=1e-14)
        assert m == 1.0


@pytest.mark.parametrize("kw,part", [
    (dict(rotary_dim=0, base=1e4), "rotary_dim"), (dict(rotary_dim=7, base=1e4), "rotary_dim"),
    (dict(rotary_dim=258, base=1e4), "rotary_dim"), (dict(rotary_dim=64, base=1.0), "base"),
    (dict(rotary_dim=64, base=math.inf), "base"), (dict(rotary_dim=64, base=math.nan), "base"),
    (dict(rotary_dim=64, base=1e4, scaling="linear", factor=0.5), "factor"),
    (dict(rotary_dim=64, base=1e4, scaling="linear", factor=math.nan), "factor"),
    (dict(rotary_dim=2, base=1e4, scaling="base", factor=2.0), "two pairs"),
    (dict(rotary_dim=64, base=1e4, scaling="bands", factor=2.0, low=1.0, high=4.0), "original_context"),
    (dict(rotary_dim=64, base=1e4, scaling="bands", factor=2.0, original_context=4096.0, low=4.0, high=4.0), "turns"),
    (dict(rotary_dim=64, base=1e4, scaling="ramp", factor=2.0, original_context=4096.0, low=0.0, high=4.0), "turns"),
    (dict(rotary_dim=64, base=1e4, scaling="pairs"), "null pointer"),
    (dict(rotary_dim=4, base=1e4, scaling="pairs", pair_factors=[1.0, 0.0]), "pair 1"),
    (dict(rotary_dim=64, base=1e4, magnitude=-1.0), "magnitude"),
    (dict(rotary_dim=64, base=1e4, scaling="other"), "scaling"),
])
def test_table_refusals(lib, kw, part):
    with pytest.raises(CudaComputeError) as e:
        paged.rope_table(**kw)
    assert e.value.code == _lib.ERR_INVALID_ARGUMENT and part in e.value.msg


def test_pair_factor_count(lib):
    with pytest.raises(CudaComputeError) as e:
        paged.rope_table(64, 1e4, scaling="pairs", pair_factors=[1.0] * 31)
    assert e.value.code == _lib.ERR_SHAPE_MISMATCH


# Addresses that are never followed: a refusal comes before any device is touched.
P = 1 << 20


def rope(**kw):
    d = dict(x=P, out=2 * P, positions=P, inv_freq=P, x_row_stride=256, x_head_stride=64, out_row_stride=256, out_head_stride=64,
             rows=2, heads=4, head_dim=64, rotary_dim=64, pairing=0, inverse=0, dtype=_lib.ROW_F32, device=0, magnitude=1.0)
    d.update(kw)
    return _lib.RopeDesc(**d)


@pytest.mark.parametrize("kw,part", [
    (dict(rows=0), "row"), (dict(heads=0), "row"), (dict(head_dim=63), "head_dim"), (dict(head_dim=258), "head_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=31), "rotary_dim"),
    (dict(pairing=2), "pairing"), (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"),
    (dict(magnitude=math.inf), "magnitude"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(positions=None), "null"),
    (dict(inv_freq=None), "null"), (dict(x=P + 2), "aligned"), (dict(out_row_stride=255), "overlap"),
    (dict(out_head_stride=0), "overlap"), (dict(out_head_stride=32), "overlap"), (dict(x_row_stride=1 << 40), "large"),
    (dict(out=P, out_row_stride=512), "in place"), (dict(positions=P + 2), "aligned"), (dict(inv_freq=P + 4), "aligned"),
])
def test_rotation_refusals(lib, kw, part):
    err = C.create_string_buffer(256)
    rc = lib.itk_rope_apply(C.byref(rope(**kw)), None, err, 256)
    assert rc == _lib.ERR_INVALID_ARGUMENT and part in err.value.decode()


def test_a_rotation_names_the_missing_descriptor_and_survives_no_buffer(lib):
    assert lib.itk_rope_apply(None, None, None, 0) == _lib.ERR_INVALID_ARGUMENT
    err = C.create_string_buffer(4)
    assert lib.itk_rope_apply(C.byref(rope(rows=0)), None, err, 4) == _lib.ERR_INVALID_ARGUMENT
    assert len(err.value) == 3  # cut, and ended


def kv(**kw):
    d = dict(k=P, v=2 * P, page_stride=16 * 2 * 64, head_stride=16 * 64, row_stride=64, n_pages=4, page_size=16, kv_heads=2, head_dim=64,
             dtype=_lib.ROW_F16, device=0)
    d.update(kw)
    return _lib.PagedKv(**d)


def batch(**kw):
    d = dict(table=P, row_start=P, kv_len=P, status=None, n_seqs=2, table_width=2, table_stride=2, total_rows=5)
    d.update(kw)
    return _lib.PagedBatch(**d)


def append(**kw):
    d = dict(q=P, q_out=P, k_new=P, v_new=P, inv_freq=P, q_row_stride=256, q_out_row_stride=256, k_row_stride=128, v_row_stride=128,
             q_heads=4, rotary_dim=64, pairing=1, dtype=_lib.ROW_F32, magnitude=1.0)
    d.update(kw)
    return _lib.PagedAppendDesc(**d)


def attention(**kw):
    d = dict(q=P, out=P, lse=None, workspace=P, workspace_bytes=1 << 40, q_row_stride=256, out_row_stride=256, q_heads=4, max_rows=1,
             window=0, dtype=_lib.ROW_F32, scale=0.125)
    d.update(kw)
    return _lib.PagedAttentionDesc(**d)


POOL = [
    (dict(kv_heads=0), _lib.ERR_ZERO_DIMENSION, "num_kv_heads"), (dict(head_dim=0), _lib.ERR_ZERO_DIMENSION, "head_dim"),
    (dict(n_pages=0), _lib.ERR_ZERO_DIMENSION, "n_pages"), (dict(head_dim=68), None, "multiple of 8"),
    (dict(head_dim=264, row_stride=264), None, "multiple of 8"), (dict(page_size=0), None, "power of two"),
    (dict(page_size=24), None, "power of two"), (dict(page_size=1 << 17), None, "power of two"), (dict(dtype=_lib.ROW_F32), None, "pages hold"),
    (dict(k=None), None, "null"), (dict(v=P + 8), None, "16-byte"), (dict(row_stride=65), None, "multiples of 8"),
    (dict(n_pages=1 << 31), None, "n_pages"), (dict(row_stride=56), None, "overlap"), (dict(head_stride=15 * 64), None, "overlap"), (dict(page_stride=31 * 64), None, "overlap"),
]
BATCH = [
    (dict(table=None), None, "null"), (dict(row_start=None), None, "null"), (dict(kv_len=None), None, "null"),
    (dict(n_seqs=0), _lib.ERR_ZERO_DIMENSION, "n_seqs"), (dict(n_seqs=1025), _lib.ERR_CAPACITY, "sequences"),
    (dict(table_width=0), _lib.ERR_ZERO_DIMENSION, "table_width"), (dict(table_stride=1), None, "table_stride"),
    (dict(total_rows=1 << 31), None, "total_rows"), (dict(table=P + 2), None, "aligned"), (dict(row_start=P + 1), None, "aligned"),
    (dict(kv_len=P + 2), None, "aligned"), (dict(status=P + 2), None, "aligned"),
]


@pytest.mark.parametrize("call", ["append", "attention"])
@pytest.mark.parametrize("which,kw,code,part", [("kv",) + c for c in POOL] + [("batch",) + c for c in BATCH])
def test_pool_and_batch_refusals(lib, call, which, kw, code, part):
    err = C.create_string_buffer(256)
    k, b = (kv(**kw), batch()) if which == "kv" else (kv(), batch(**kw))
    fn, d = (lib.itk_paged_append, append()) if call == "append" else (lib.itk_paged_attention, attention())
    rc = fn(C.byref(k), C.byref(b), C.byref(d), None, err, 256)
    assert rc == (code or _lib.ERR_INVALID_ARGUMENT) and part in err.value.decode(), err.value


@pytest.mark.parametrize("kw,part", [
    (dict(k_new=None), "null"), (dict(v_new=None), "null"), (dict(q_out=None), "go together"), (dict(q=None), "go together"),
    (dict(q_heads=0), "go together"), (dict(rotary_dim=33), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"), (dict(pairing=2), "pairing"),
    (dict(magnitude=math.nan), "magnitude"), (dict(dtype=_lib.ROW_BF16), "bf16 rows"), (dict(dtype=9), "element type"),
    (dict(k_new=P + 1), "aligned"), (dict(inv_freq=P + 4), "aligned"), (dict(q_out_row_stride=255), "overlap"), (dict(q_row_stride=512), "in place"),
])
def test_append_refusals(lib, kw, part):
    err = C.create_string_buffer(256)
    rc = lib.itk_paged_append(C.byref(kv()), C.byref(batch()), C.byref(append(**kw)), None, err, 256)
    assert rc == _lib.ERR_INVALID_ARGUMENT and part in err.value.decode(), err.value


@pytest.mark.parametrize("kw,code,part", [
    (dict(q_heads=0), _lib.ERR_ZERO_DIMENSION, "num_q_heads"), (dict(q_heads=3), _lib.ERR_NON_DIVISIBLE_HEADS, "divide evenly"),
    (dict(q=None), None, "null"), (dict(out=None), None, "null"), (dict(workspace=None), None, "null"), (dict(workspace=P + 16), None, "256-byte"),
    (dict(q=P + 8), None, "16-byte"), (dict(lse=P + 2), None, "aligned"), (dict(scale=math.nan), None, "scale"), (dict(q_row_stride=260), None, "multiples of 8"),
    (dict(out_row_stride=248), None, "overlap"), (dict(dtype=_lib.ROW_BF16), None, "bf16 rows"),
])
def test_attention_refusals(lib, kw, code, part):
    err = C.create_string_buffer(256)
    rc = lib.itk_paged_attention(C.byref(kv()), C.byref(batch()), C.byref(attention(**kw)), None, err, 256)
    assert rc == (code or _lib.ERR_INVALID_ARGUMENT) and part in err.value.decode(), err.value


@pytest.mark.parametrize("kw,part", [(dict(q_heads=65536), "q_heads"), (dict(q_heads=1 << 30), "q_heads"), (dict(scale=3e38), "scale"), (dict(scale=-math.inf), "scale")])
def test_attention_refuses_what_its_kernels_cannot_count(lib, kw, part):
    """Heads whose channels would pass 32 bits, and a scale that is infinite in the base the kernels work in."""
    err = C.create_string_buffer(256)
    rc = lib.itk_paged_attention(C.byref(kv()), C.byref(batch(total_rows=1)), C.byref(attention(**kw)), None, err, 256)
    assert rc == _lib.ERR_INVALID_ARGUMENT and part in err.value.decode(), err.value


@pytest.mark.parametrize("name", ["itk_paged_append", "itk_paged_attention"])
def test_sizes_that_their_fields_cannot_hold_are_refused_by_name(name, monkeypatch):
    """A table whose rows lie 2^33 elements apart, and one whose only row does (nothing is stepped over)."""
    packed = []
    monkeypatch.setattr(paged, "_calls", {name: lambda *args: packed.append(_lib.PagedBatch.from_buffer_copy(args[1])) or _lib.OK})
    monkeypatch.setattr(paged, "_written", lambda ts: None)
    kv = paged.PagedKv.__new__(paged.PagedKv)
    kv._index, kv.head_dim, kv.kv_heads, kv._kv, kv._scale = 0, 64, 2, b"", 0.125
    kv.k = kv.v = x = OnCard(torch.zeros(4, 2, 64))
    ws = OnCard(torch.zeros(8, dtype=torch.uint8))

    def call(n):
        table = OnCard(torch.zeros(n, 3, dtype=torch.int32))
        table.stride = lambda: (1 << 33, 1)
        batch = (table, OnCard(torch.zeros(n + 1, dtype=torch.int32)), OnCard(torch.zeros(n, dtype=torch.int32)))
        return kv.append(x, x, *batch, stream=7) if name == "itk_paged_append" else kv.attention(x, *batch, max_rows=1, out=x, workspace=ws, stream=7)

    with pytest.raises(CudaComputeError) as e:
        call(2)
    assert "out of range" in e.value.msg and not packed
    call(1)
    assert packed[0].table_stride == packed[0].table_width == 3


def test_too_many_pairs(lib):
    err = C.create_string_buffer(256)
    rc = lib.itk_paged_attention(C.byref(kv()), C.byref(batch(total_rows=1 << 30)), C.byref(attention()), None, err, 256)
    assert rc == _lib.ERR_INVALID_ARGUMENT and "total_rows" in err.value.decode()


def test_missing_descriptors(lib):
    for fn in (lib.itk_paged_append, lib.itk_paged_attention):
        assert fn(None, None, None, None, None, 0) == _lib.ERR_INVALID_ARGUMENT
        assert fn(C.byref(kv()), None, None, None, None, 0) == _lib.ERR_INVALID_ARGUMENT
        assert fn(C.byref(kv()), C.byref(batch()), None, None, None, 0) == _lib.ERR_INVALID_ARGUMENT


def test_wait_limits(lib):
    for bad in (-1, (1 << 22) + 1, 1 << 32):
        with pytest.raises(CudaComputeError) as e:
            paged.wait_limit(bad)
        assert e.value.code == _lib.ERR_INVALID_ARGUMENT
    for fine in (1, 1 << 22, 0):
        paged.wait_limit(fine)


class OnCard:
    """Stands in for a tensor on a device that is not there, as far as the calls look at it."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


def calls_on_card():
    """The three calls on stand-ins, by the name of their entry point: call(**tensors), and the tensors it writes."""
    i32 = lambda *shape: OnCard(torch.zeros(*shape, dtype=torch.int32))
    f = OnCard(torch.zeros(32, dtype=torch.float64))
    kv = paged.PagedKv.__new__(paged.PagedKv)
    kv._index, kv.head_dim, kv.kv_heads, kv._kv, kv._scale = 0, 64, 2, b"", 0.125
    rows = {n: OnCard(torch.zeros(4, 2, 64)) for n in ("x", "out", "q", "q_out", "k", "v", "k_pool", "v_pool")}
    rows["lse"] = OnCard(torch.zeros(4, 2))
    kv.k, kv.v = rows["k_pool"], rows["v_pool"]
    batch, ws = (i32(1, 3), i32(2), i32(1)), OnCard(torch.zeros(8, dtype=torch.uint8))
    return rows, {
        "itk_rope_apply": (lambda: paged.rope_apply(rows["x"], i32(4), f, out=rows["out"], stream=7), ["out"], ["x", "out"]),
        "itk_paged_append": (lambda: kv.append(rows["k"], rows["v"], *batch, q=rows["q"], q_out=rows["q_out"], inv_freq=f, stream=7),
                             ["k_pool", "v_pool", "q_out"], ["k", "v", "q", "q_out", "k_pool", "v_pool"]),
        "itk_paged_attention": (lambda: kv.attention(rows["q"], *batch, max_rows=4, out=rows["out"], lse=rows["lse"], workspace=ws, stream=7),
                                ["out", "lse"], ["q", "out", "lse", "k_pool", "v_pool"]),
    }


@pytest.mark.parametrize("name", ["itk_rope_apply", "itk_paged_append", "itk_paged_attention"])
def test_tensors_that_require_a_gradient_are_refused_while_gradients_are_enabled(name, monkeypatch):
    made, written = [], []
    monkeypatch.setattr(paged, "_calls", {name: lambda *args: made.append(name) or _lib.OK})
    monkeypatch.setattr(paged, "_written", lambda ts: written.extend(ts))
    rows, calls = calls_on_card()
    call, writes, takes = calls[name]
    call()
    assert made == [name] and written == [rows[n] for n in writes]
    for n in takes:
        rows[n].t.requires_grad_()
        with pytest.raises(CudaComputeError) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARGUMENT and "gradient" in e.value.msg and len(made) == 1
        rows[n].t.requires_grad_(False)
    for n in takes:
        rows[n].t.requires_grad_()
    with torch.no_grad():
        call()
    assert len(made) == 2


@pytest.mark.parametrize("name", ["itk_rope_apply", "itk_paged_append", "itk_paged_attention"])
def test_a_failed_call_is_made_once(lib, name, monkeypatch):
    """A call that reports an error may have run (an asynchronous launch before it failed): it is not made again, and its
    reason is the one it gave."""
    made = []

    def entry(*args):
        made.append(args)
        C.memmove(args[-2], b"launch failed: something before it\0", 35)
        return _lib.ERR_CUDA if len(made) == 1 else _lib.OK

    monkeypatch.setattr(paged, "_calls", {name: entry})
    monkeypatch.setattr(paged, "_written", lambda ts: None)
    call = calls_on_card()[1][name][0]
    with pytest.raises(CudaComputeError) as e:
        call()
    assert e.value.code == _lib.ERR_CUDA and e.value.msg == "launch failed: something before it"
    assert len(made) == 1
    call()
    assert len(made) == 2


@pytest.mark.parametrize("name,args", [("itk_rope_apply", 1), ("itk_paged_append", 3), ("itk_paged_attention", 3)])
def test_the_library_writes_its_reason_where_the_call_says(lib, name, args):
    assert paged._entry(name, args)(*[None] * args, None, paged._reason.at, 256) == _lib.ERR_INVALID_ARGUMENT
    with pytest.raises(CudaComputeError) as e:
        paged._reason.refuse(_lib.ERR_INVALID_ARGUMENT)
    assert "null pointer" in e.value.msg
