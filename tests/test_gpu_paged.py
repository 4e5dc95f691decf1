"""The paged operators on the device against their definitions in 64 bits (``pagedref``), with tolerances derived there."""
import ctypes as C
import math
import threading

import numpy as np
import pytest
import torch

from itak_torch_rebuild_b200 import CudaCompute, CudaComputeError, KvDtype, _lib, paged
from pagedref import PAGE, U, Batch, DeviceBatch, attend, attend_bound, plan_stream, plan_tc, rotate, rotation_bound, within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
NAN = math.nan


def table(rot, dev="cuda", **kw):
    f, m = paged.rope_table(rot, 10000.0, **kw)
    return f, torch.from_numpy(f).to(dev), m


# ---- rotation ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("rows,heads,d,rot", [(1, 1, 2, 2), (3, 5, 64, 64), (7, 3, 96, 32), (2, 33, 128, 128), (5, 2, 80, 62),
                                              (4, 2, 256, 256), (2, 2, 10, 6), (1, 64, 128, 48), (2, 300, 64, 2)])
def test_rotation(t, pairing, rows, heads, d, rot):
    g = torch.Generator().manual_seed(rows * 100 + d)
    x = torch.randn(rows, heads, d, generator=g).to(t)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    pos[0] = 0
    f, fd, _ = table(rot)
    got = paged.rope_apply(x.cuda(), pos.cuda(), fd, pairing=pairing, magnitude=1.25)
    extra, _ = rotation_bound(x, f, pairing, 1.25, t)
    within(got, rotate(x, pos, f, pairing, 1.25), extra, t)
    if rot < d:
        assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    inplace = x.cuda()
    assert paged.rope_apply(inplace, pos.cuda(), fd, pairing=pairing, magnitude=1.25, out=inplace) is inplace
    assert torch.equal(inplace, got)


def test_rotation_at_position_zero_and_far_away():
    f, fd, _ = table(128)
    x = torch.randn(4, 2, 128)
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1], dtype=torch.int32)
    got = paged.rope_apply(x.cuda(), pos.cuda(), fd)
    assert torch.equal(got[0].cpu(), x[0])
    extra, _ = rotation_bound(x, f, 0, 1.0, F32)
    # an f64 product p * f is off by 2^-53 of up to 2^31 radians, on both sides: 2^-21 of the pair
    size = x.double().abs().sum(-1, keepdim=True)
    within(got, rotate(x, pos, f, 0), extra + 2.0 ** -21 * size, F32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pairing", [0, 1])
def test_rotation_of_strided_rows(t, pairing):
    """Q inside a projection's output; heads outermost; rows that sixteen-byte words cannot address; a broadcast row."""
    f, fd, _ = table(64)
    pos = torch.arange(5, dtype=torch.int32) * 77
    whole = torch.randn(5, 9, 64).to(t).cuda()
    out = torch.full((5, 9, 64), NAN, dtype=t, device="cuda")
    views = [(whole[:, 2:6], out[:, 2:6]), (whole.transpose(0, 1).contiguous().transpose(0, 1)[:, :4], torch.empty(4, 5, 64, dtype=t, device="cuda").transpose(0, 1)),
             (torch.randn(5, 4, 67).to(t).cuda()[..., 1:65], torch.empty(5, 4, 66, dtype=t, device="cuda")[..., :64]),
             (whole[:1].expand(5, 9, 64)[:, 3:7], torch.empty(5, 4, 64, dtype=t, device="cuda"))]
    for x, o in views:
        paged.rope_apply(x, pos.cuda(), fd, pairing=pairing, out=o)
        extra, _ = rotation_bound(x.cpu(), f, pairing, 1.0, t)
        within(o, rotate(x.cpu(), pos, f, pairing), extra, t)
    assert bool(torch.isnan(out[:, :2]).all()) and bool(torch.isnan(out[:, 6:]).all())


@pytest.mark.parametrize("pairing", [0, 1])
def test_gradient_against_the_formula_and_differences(pairing):
    f, fd, m = table(24, scaling="ramp", factor=4.0, original_context=512.0, low=1.0, high=32.0)
    x, gy = torch.randn(3, 2, 40), torch.randn(3, 2, 40)
    pos = torch.tensor([5, 900, 0], dtype=torch.int32)
    got = paged.rope_apply(gy.cuda(), pos.cuda(), fd, pairing=pairing, magnitude=m, inverse=True)
    xa = x.double().requires_grad_()
    a = torch.arange(12) * (2 if pairing == 0 else 1)
    b = a + (1 if pairing == 0 else 12)
    ang = pos.double()[:, None, None] * torch.from_numpy(f)
    y0, y1 = m * (xa[..., a] * ang.cos() - xa[..., b] * ang.sin()), m * (xa[..., a] * ang.sin() + xa[..., b] * ang.cos())
    loss = (y0 * gy.double()[..., a]).sum() + (y1 * gy.double()[..., b]).sum() + (xa[..., 24:] * gy.double()[..., 24:]).sum()
    loss.backward()
    extra, _ = rotation_bound(gy, f, pairing, m, F32)
    within(got, xa.grad, extra, F32)
    # differences: the map is linear, so f(x + e) - f(x) = f(e) up to rounding; one entry of every kind of channel
    def value(z):
        return float((paged.rope_apply(z.cuda(), pos.cuda(), fd, pairing=pairing, magnitude=m).double().cpu() * gy.double()).sum())
    for r, h, c in [(0, 0, 0), (1, 1, 1), (1, 0, 13), (2, 1, 23), (0, 1, 39)]:
        e = torch.zeros_like(x)
        e[r, h, c] = 0.5
        # two outputs of size <= 1.5 m |x + e| each rounded in f32, on both sides, times |gy|
        slack = 8 * 16 * 2.0 ** -24 * m * float((x.abs().max() + 0.5) * gy.abs().max())
        assert abs((value(x + e) - value(x - e)) - float(got[r, h, c])) <= slack


def test_rotation_refuses_on_the_python_side():
    f, fd, _ = table(64)
    x, pos = torch.randn(4, 2, 64).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    for bad in (dict(positions=pos.long()), dict(positions=pos[:3]), dict(inv_freq=fd.float()), dict(x=x.double()), dict(x=x.cpu()),
                dict(out=torch.empty(4, 2, 64, dtype=F16, device="cuda")), dict(out=x[:2]), dict(inv_freq=torch.zeros(0, dtype=torch.float64, device="cuda")),
                dict(x=x[..., ::2]), dict(x=x[:0], positions=pos[:0])):
        kw = dict(x=x, positions=pos, inv_freq=fd)
        kw.update(bad)
        with pytest.raises(CudaComputeError):
            paged.rope_apply(kw.pop("x"), kw.pop("positions"), kw.pop("inv_freq"), **kw)


def leave_an_error_behind(how):
    lib = _lib.load()
    if how == "a device that is not there":
        assert lib.itk_paged_attention_workspace(torch.cuda.device_count() + 7) == 0
    elif how == "a call on a device that is not there":
        d = _lib.RopeDesc(1 << 20, 1 << 21, 1 << 20, 1 << 20, 64, 64, 64, 64, 1, 1, 64, 64, 0, 0, _lib.ROW_F32, torch.cuda.device_count() + 7, 1.0)
        assert lib.itk_rope_apply(C.byref(d), None, None, 0) == _lib.ERR_CUDA
    else:  # 8 TiB of slots
        with pytest.raises(CudaComputeError):
            CudaCompute(8, 8, 8, 128, n_slots=64, max_context=1 << 22, chunk_cap=8, kv_dtype=KvDtype.F32)


@pytest.mark.parametrize("how", ["a device that is not there", "a call on a device that is not there", "a cache that does not fit"])
def test_an_earlier_error_does_not_turn_rows_twice(how):
    """A refused call of this library before one that rotates in place: the rows are turned once, and nothing is raised."""
    f, fd, _ = table(64)
    x, pos = torch.randn(4, 2, 64), torch.tensor([3, 50, 700, 9000], dtype=torch.int32)
    extra, _ = rotation_bound(x, f, 0, 1.0, F32)
    y = x.cuda()
    leave_an_error_behind(how)
    paged.rope_apply(y, pos.cuda(), fd, out=y)
    within(y, rotate(x, pos, f, 0), extra, F32)
    b = Batch([4], [9], 2, 1, 64, F32, 8, "head")
    q, k = x.cuda(), torch.randn(4, 1, 64).cuda()
    leave_an_error_behind(how)
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, q=q, q_out=q, inv_freq=fd)
    within(q, rotate(x, [5, 6, 7, 8], f, 0), extra, F32)


# ---- append -----------------------------------------------------------------------------------------------------------


def check_append(b, k, v, q, f, pairing, q_out, status=None):
    """Every page row is either one of the batch's new rows or untouched."""
    pt = PAGE[b.t]
    want_k, want_v = b.k_h.clone(), b.v_h.clone()
    seen = torch.zeros(b.n_pages, b.page, dtype=torch.bool)
    for s, (r, n) in enumerate(zip(b.rows, b.lens)):
        lo = b.starts[s]
        for i in range(r):
            p = n - r + i
            page = int(b.table_h[s, p // b.page]) if p >= 0 else -1
            if p < 0 or not 0 <= page < b.n_pages:
                continue
            seen[page, p % b.page] = True
            for pool, src, turned in ((b.k, k, True), (b.v, v, False)):
                row = src[lo + i].cpu()
                got = b.cell(pool.cpu(), page, p % b.page)
                if turned and f is not None:
                    extra, _ = rotation_bound(row[None], f, pairing, 1.0, pt)
                    within(got[None], rotate(row[None], [p], f, pairing), extra, pt)
                    assert torch.equal(got[..., 2 * len(f):], row[..., 2 * len(f):].to(pt))
                else:
                    assert torch.equal(got, row.to(pt))
        if q is not None and r:
            keep = [i for i in range(r) if n - r + i >= 0]
            if keep:
                rows = q[lo:lo + r].cpu()[keep]
                pos = [n - r + i for i in keep]
                if f is None:
                    assert torch.equal(q_out[lo:lo + r].cpu()[keep], rows)
                else:
                    extra, _ = rotation_bound(rows, f, pairing, 1.0, b.t)
                    within(q_out[lo:lo + r].cpu()[keep], rotate(rows, pos, f, pairing), extra, b.t)
    for pool, was in ((b.k.cpu(), want_k), (b.v.cpu(), want_v)):
        by_row = pool.transpose(1, 2) if b.layout == "head" else pool
        was = was.transpose(1, 2) if b.layout == "head" else was
        assert torch.equal(by_row[~seen].view(torch.int16), was[~seen].view(torch.int16)), "a row outside the batch was written"


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pairing,rot", [(0, 64), (1, 64), (1, 32), (0, 6), (1, 6), (0, 0)])
@pytest.mark.parametrize("layout,page", [("head", 16), ("token", 8), ("head", 1), ("token", 64)])
def test_append(t, pairing, rot, layout, page):
    b = Batch([1, 0, 9, 3, 20], [1, 5, 9, 40, 21], 6, 2, 64, t, page, layout, extra_rows=3)
    qkv = torch.randn(b.total, 10, 64).to(t).cuda()
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    f, fd, _ = table(rot) if rot else (None, None, 1.0)
    q_out = torch.full((b.total, 6, 64), 7.0, dtype=t, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    b.k_h, b.v_h = b.k.cpu(), b.v.cpu()
    b.cell_was = None
    assert b and PagedOf(b).append(k, v, b.table, b.row_start, b.kv_len, q=q, q_out=q_out, inv_freq=fd, pairing=pairing, status=status) is q_out
    check_append(b, k, v, q, f, pairing, q_out)
    assert int(status) == 0 and bool((q_out[b.starts[-1]:] == 7.0).all())


def PagedOf(b):
    return paged.PagedKv(b.k, b.v, layout=b.layout)


@pytest.mark.parametrize("d,hkv", [(8, 1), (128, 8), (256, 3), (72, 5)])
def test_append_without_q_and_other_widths(d, hkv):
    b = Batch([4, 2], [30, 2], hkv, hkv, d, F32, 16, "token")
    k, v = torch.randn(b.total, hkv, d).cuda(), torch.randn(b.total, hkv, d).cuda()
    f, fd, _ = table(min(d, 8))
    b.k_h, b.v_h = b.k.cpu(), b.v.cpu()
    assert PagedOf(b).append(k, v, b.table, b.row_start, b.kv_len, inv_freq=fd, pairing=1) is None
    check_append(b, k, v, None, f, 1, None)


def test_append_keeps_bits_of_what_it_does_not_rotate():
    """V and the channels behind the rotated part: infinities, NaN and signed zeros as they came (f32 NaN as an append
    stores it: sign | 0x7e00)."""
    for t in TYPES:
        b = Batch([2], [2], 1, 1, 16, t, 8, "head")
        odd = torch.tensor([math.inf, -math.inf, NAN, -0.0, 0.0, 65504.0, 1e-7, -1e-8, 1.0, 2.0, 3.0, 70000.0, -70000.0, 5.0, 6.0, 7.0])
        v = odd.to(t).repeat(2, 1, 1).cuda()
        _, fd, _ = table(8)
        PagedOf(b).append(v, v, b.table, b.row_start, b.kv_len, inv_freq=fd)
        page = int(b.table_h[0, 0])
        want = odd.to(t).to(PAGE[t])
        got_v, got_k = b.v.cpu()[page, 0, 0], b.k.cpu()[page, 0, 0]
        for got, part in ((got_v, slice(0, 16)), (got_k, slice(8, 16))):
            fine = ~torch.isnan(want[part])
            assert torch.equal(got[part][fine].view(torch.int16), want[part][fine].view(torch.int16))
            assert bool(torch.isnan(got[part][~fine]).all())


def test_append_drops_what_the_pool_does_not_hold():
    """A page number outside the pool, a sequence longer than its table, rows before position 0, starts that run backwards:
    reported, nothing else touched."""
    b = Batch([3, 2, 2], [20, 8, 40], 2, 1, 16, F16, 8, "head")
    b.table[1, 0] = b.n_pages  # one past the end
    b.table_h[1, 0] = b.n_pages
    k = torch.randn(b.total, 1, 16).half().cuda()
    b.k_h, b.v_h = b.k.cpu(), b.v.cpu()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, status=status)
    assert int(status) == 1
    check_append(b, k, k, None, None, 0, None)

    b = Batch([3, 2], [20, 2], 2, 1, 16, F16, 8, "head")
    k = torch.randn(b.total, 1, 16).half().cuda()
    b.kv_len[0], b.kv_len[1] = 1000, 1  # longer than the table; two new rows in one key
    before = b.k.clone()
    status.zero_()
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, status=status)
    assert int(status) == 2 | 4
    b.kv_len[0], b.kv_len[1] = 20, 2
    b.row_start.copy_(torch.tensor([3, 0, 5]))
    status.zero_()
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, status=status)
    assert int(status) & 8
    b.row_start.copy_(torch.tensor([0, 3, 1000]))
    status.zero_()
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, status=status)
    assert int(status) & 8
    assert before.shape == b.k.shape


def rows_of(b, pool):
    """A pool's bits as [page][row][heads][D], on the host."""
    pool = pool.cpu().view(torch.int16)
    return (pool.transpose(1, 2) if b.layout == "head" else pool).clone()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pairing,rot,lead", [(0, 0, 0), (1, 32, 0), (1, 6, 0), (0, 16, 1)])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_rows_behind_the_table_are_dropped_where_they_stand(t, pairing, rot, lead, layout):
    """A sequence longer than its row of the table: positions go by the stated length, the rows that still have a place are
    stored there, the others nowhere - least of all over the keys before them.  Queries are turned at their positions.
    ``lead``: rows that start off a 16-byte boundary."""
    d, page = 32, 8
    b = Batch([3, 3, 2, 1], [24, 24, 24, 24], 4, 2, d, t, page, layout)
    stated = [26, 1000, 24, -1]
    b.kv_len.copy_(torch.tensor(stated))
    f, fd, _ = table(rot) if rot else (None, None, 1.0)
    wide = torch.randn(b.total, 8 * d + lead).to(t).cuda()
    qkv = wide[:, lead:].unflatten(1, (8, d))
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    want_k, want_v = rows_of(b, b.k), rows_of(b, b.v)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = PagedOf(b).append(k, v, b.table, b.row_start, b.kv_len, q=q, inv_freq=fd, pairing=pairing, status=status)
    assert int(status) == 2
    got_k, got_v = rows_of(b, b.k), rows_of(b, b.v)
    for s, i, p in ((0, 0, 23), (2, 0, 22), (2, 1, 23)):
        row, at, off = b.starts[s] + i, int(b.table_h[s, p // page]), p % page
        assert torch.equal(got_v[at, off], v[row].cpu().to(PAGE[t]).view(torch.int16))
        if rot:
            extra, _ = rotation_bound(k[row:row + 1].cpu(), f, pairing, 1.0, PAGE[t])
            within(got_k[at, off].view(PAGE[t])[None], rotate(k[row:row + 1].cpu(), [p], f, pairing), extra, PAGE[t])
        else:
            assert torch.equal(got_k[at, off], k[row].cpu().to(PAGE[t]).view(torch.int16))
        want_k[at, off], want_v[at, off] = got_k[at, off], got_v[at, off]
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v), "a row outside the batch was written"
    for s in (0, 1, 2):
        lo, r = b.starts[s], b.rows[s]
        if rot:
            extra, _ = rotation_bound(q[lo:lo + r].cpu(), f, pairing, 1.0, t)
            within(q_out[lo:lo + r], rotate(q[lo:lo + r].cpu(), [stated[s] - r + i for i in range(r)], f, pairing), extra, t)
        else:
            assert torch.equal(q_out[lo:lo + r], q[lo:lo + r])


@pytest.mark.parametrize("starts,lens,bits,kept", [
    ([0, 3, 5], [1000, 1], 2 | 4, [(1, 4, 0)]),                 # (sequence, packed row, position)
    ([3, 0, 5], [20, 2], 4 | 8, [(1, 3, 0), (1, 4, 1)]),
    ([0, 3, 1000], [20, 2], 8, [(0, 0, 17), (0, 1, 18), (0, 2, 19), (1, 3, 0), (1, 4, 1)]),
    ([7, 7, 7], [20, 2], 8, []),
    ([0, 3, 5], [2 ** 31 - 1, 24], 2, [(1, 3, 22), (1, 4, 23)]),
])
def test_append_of_malformed_batches_writes_what_belongs(starts, lens, bits, kept):
    b = Batch([3, 2], [24, 24], 2, 1, 16, F16, 8, "head")
    k = torch.randn(b.total, 1, 16).half().cuda()
    want = [rows_of(b, b.k), rows_of(b, b.v)]
    b.row_start.copy_(torch.tensor(starts))
    b.kv_len.copy_(torch.tensor(lens))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len, status=status)
    assert int(status) == bits
    for s, row, p in kept:
        for pool in want:
            pool[int(b.table_h[s, p // 8]), p % 8] = k[row].cpu().view(torch.int16)
    assert torch.equal(rows_of(b, b.k), want[0]) and torch.equal(rows_of(b, b.v), want[1])


# ---- attention --------------------------------------------------------------------------------------------------------


def run_attention(b, window=0, scale=None, **kw):
    out = torch.full((b.total, b.hq, b.d), 7.0, dtype=b.t, device="cuda")
    lse = torch.full((b.total, b.hq), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = paged.attention_workspace("cuda:0")
    n_tickets = 4 * 2 * torch.cuda.get_device_properties(0).multi_processor_count
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=max(b.rows), window=window, scale=scale, out=out, lse=lse,
                         status=status, workspace=ws, **kw)
    b.check(out, lse, scale, window)
    assert int(status) == 0
    assert bool((ws[:n_tickets] == 0).all()), "the workspace's tickets are not zero again"
    assert bool((out[b.starts[-1]:] == 7.0).all()) and bool((lse[b.starts[-1]:] == 7.0).all())
    return out, lse


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 1, 128), (3, 3, 128), (2, 1, 96), (14, 2, 128), (2, 2, 256), (5, 1, 8), (32, 2, 64), (17, 1, 80)])
@pytest.mark.parametrize("layout,page", [("head", 16), ("token", 32)])
def test_decode(t, hq, hkv, d, layout, page):
    run_attention(Batch([1] * 6, [1, 16, 17, 64, 65, 301], hq, hkv, d, t, page, layout, extra_rows=2))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_blocks_of_rows_over_all_page_sizes(t, page, layout):
    run_attention(Batch([7, 0, 1, 5, 33, 2], [7, 3, 100, 64, 150, 2], 6, 2, 64, t, page, layout, extra_rows=1))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (2, 2, 64), (7, 1, 64), (2, 1, 96), (2, 1, 256), (3, 1, 40)])
@pytest.mark.parametrize("rows,lens", [([129], [129]), ([64, 1, 0, 200], [300, 77, 5, 256]), ([130, 31], [130, 500])])
def test_chunks(t, hq, hkv, d, rows, lens):
    run_attention(Batch(rows, lens, hq, hkv, d, t, 16, "head", extra_rows=3))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 200, 100000, 2 ** 32 - 1])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [5, 64, 333]), ([9, 70, 140], [9, 290, 300])])
def test_windows(t, window, rows, lens):
    run_attention(Batch(rows, lens, 4, 2, 64, t, 16, "token"), window=window)


@pytest.mark.parametrize("t", TYPES)
def test_pages_behind_the_window_may_be_gone(t):
    """Pages that no row of the call can see are not followed: their table entries may hold anything."""
    for rows, n, window in ((1, 300, 40), (5, 300, 40), (100, 300, 40)):
        b = Batch([rows], [n], 4, 2, 64, t, 16, "head")
        first = n - rows - window + 1
        for j in range(first // 16):
            page = int(b.table_h[0, j])
            b.k[page], b.v[page] = NAN, NAN
            b.table[0, j] = -7
        run_attention(b, window=window)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-30])
def test_scales(t, scale):
    run_attention(Batch([1, 40], [77, 90], 4, 2, 64, t, 16, "head"), scale=scale)


@pytest.mark.parametrize("t", TYPES)
def test_large_scores_rescale_the_accumulator(t):
    """Maxima that keep growing along the keys: every tile raises the running maximum far beyond the lazy step."""
    for rows, n in ((1, 400), (60, 400)):
        b = Batch([rows], [n], 4, 2, 64, t, 16, "head")
        ramp = torch.linspace(0.1, 12.0, n)[:, None, None]
        q = torch.ones(b.total, 4, 64) * 0.5 + 0.01 * torch.randn(b.total, 4, 64)
        b.q_h = q.to(t)
        b.q.copy_(b.q_h)
        b.keys[0] = (torch.ones(n, 2, 64) * ramp + 0.01 * torch.randn(n, 2, 64)).to(PAGE[t])
        for p in range(n):
            b.cell(b.k, int(b.table_h[0, p // 16]), p % 16).copy_(b.keys[0][p])
        run_attention(b)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_rows_that_see_nothing(t, rows):
    """More new rows than keys: the rows before position 0 give zeros and -infinity, and are reported."""
    b = Batch([rows, 1, rows], [rows + 3, 0, rows + 9], 4, 2, 64, t, 16, "head")
    out, lse = torch.full((b.total, 4, 64), 7.0, dtype=t, device="cuda"), torch.full((b.total, 4), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows, out=out, lse=lse, status=status)
    b.check(out, lse, only=(0, 2))
    assert int(status) == 4
    gone = out[b.starts[1]:b.starts[2]]
    assert bool((gone == 0).all()) and bool((lse[b.starts[1]:b.starts[2]] == -math.inf).all())
    # and a block that reaches before the start in part
    b = Batch([rows + 5], [rows + 5], 4, 2, 64, t, 16, "head")
    b.kv_len[0] = rows
    out = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows + 5, lse=(lse := torch.empty(b.total, 4, device="cuda")))
    assert bool((out[:5] == 0).all()) and bool((lse[:5] == -math.inf).all())
    short = Batch([rows], [rows], 4, 2, 64, t, 16, "head")
    short.q_h, short.keys, short.values = b.q_h[5:], [b.keys[0][:rows]], [b.values[0][:rows]]
    short.check(out[5:], lse[5:])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [1, 50])
def test_infinite_and_nan_keys_stay_with_the_rows_that_see_them(t, rows):
    """A NaN key reaches the rows that see it, and a key of one sequence no row of another; the pool's unused rows are NaN
    throughout these tests."""
    b = Batch([rows, rows], [100, 100], 4, 2, 64, t, 16, "head")
    p = 100 - (rows + 1) // 2  # rows from this position on see it
    page = int(b.table_h[0, p // 16])
    b.cell(b.k, page, p % 16).fill_(NAN)
    out = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows)
    b.check(out, only=(1,))
    sees = torch.tensor([100 - rows + r >= p for r in range(rows)])
    bad = torch.isnan(out[:rows]).all(-1).all(-1).cpu()
    assert bool(bad[sees].all()) and not bool(torch.isnan(out[:rows].cpu()[~sees]).any())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_page_numbers_outside_the_pool_are_reported_and_not_followed(t, rows):
    b = Batch([rows, rows], [200, 120], 4, 2, 64, t, 16, "head")
    b.table[0, 3] = b.n_pages
    b.table[0, 5] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows, status=status)
    assert int(status) == 1
    b.check(out, only=(1,))
    # their keys read as zeros
    for s in (3, 5):
        b.keys[0][16 * s:16 * s + 16] = 0
        b.values[0][16 * s:16 * s + 16] = 0
    b.check(out, only=(0,))


@pytest.mark.parametrize("rows", [1, 40])
def test_malformed_batches_are_cut_and_reported(rows):
    b = Batch([rows, rows], [100, 90], 4, 2, 64, F16, 16, "head")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = lambda: (b.q, b.table, b.row_start, b.kv_len)
    b.kv_len[1] = 2 ** 31 - 1
    PagedOf(b).attention(*args(), max_rows=rows, status=status)
    assert int(status) & 2
    b.kv_len[1] = 90
    status.zero_()
    b.row_start.copy_(torch.tensor([rows, 0, 2 * rows]))
    PagedOf(b).attention(*args(), max_rows=rows, status=status)
    assert int(status) & 8
    status.zero_()
    b.row_start.copy_(torch.tensor([0, rows, 1 << 30]))
    out = PagedOf(b).attention(*args(), max_rows=rows, status=status)
    assert int(status) & 8
    b.check(out)  # cut to the rows there are


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [1, 7, 150])
@pytest.mark.parametrize("over", [1, 5, 70, 10 ** 9])
@pytest.mark.parametrize("window", [0, 3, 66, 200])
def test_attention_of_a_sequence_longer_than_its_table(t, rows, over, window):
    """Positions go by the stated length; the keys behind the table's last column are not there."""
    room = 240
    b = Batch([rows, 2], [room, 90], 4, 2, 64, t, 16, "head")
    b.kv_len[0] = room + over
    out, lse = torch.full((b.total, 4, 64), 7.0, dtype=t, device="cuda"), torch.full((b.total, 4), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows, window=window, out=out, lse=lse, status=status)
    assert int(status) == 2
    b.check(out, lse, window=window, only=(1,))
    scale = float(np.float32(1.0 / math.sqrt(b.d)))
    for r in range(rows):
        p = room + over - rows + r
        behind = max(0, p - (room - 1))  # a row that stands behind the last key sees what one at the last key would, less that
        got, got_lse = out[r:r + 1], lse[r:r + 1].double().cpu()
        if window and window <= behind:
            assert bool((got == 0).all()) and bool((got_lse == -math.inf).all())
            continue
        want, want_lse, mean, slack = attend(b.q_h[r:r + 1].double(), b.keys[0].double(), b.values[0].double(), p - behind, scale,
                                             window - behind if window else 0)
        within(got, want, attend_bound(mean, slack, room, b.d, t), t)
        tol = (b.d + 16) * 2.0 ** -24 * slack + 2.0 ** -20 * slack + (room / 16 + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * want_lse.abs()
        assert bool(((got_lse - want_lse).abs() <= tol).all())


def test_a_wrong_bound_of_the_rows_changes_nothing_but_the_kernel():
    b = Batch([40, 1], [100, 300], 8, 2, 128, BF16, 16, "head")
    for bound in (0, 1, 17, 10 ** 6):
        out = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=bound)
        b.check(out)


@pytest.mark.parametrize("n,rows", [(1024, 1), (1000, 3), (300, 20)])
def test_many_sequences(n, rows):
    rng = np.random.default_rng(n)
    lens = rng.integers(rows, 60, n).tolist()
    r = [int(x) for x in rng.integers(0, rows + 1, n)]
    b = Batch(r, lens, 2, 1, 64, BF16, 16, "token")
    run_attention(b)


@pytest.mark.parametrize("t", TYPES)
def test_strided_rows_and_pages(t):
    """Q and out inside wider rows, pools that are slices of a layer-major allocation, a table with spare columns."""
    b = Batch([1, 12], [90, 60], 4, 2, 64, t, 16, "head", width=9)
    pools = torch.full((b.n_pages, 3, 2, 2, 16, 64), NAN, dtype=PAGE[t], device="cuda")  # [page][layer][K, V][head][row][D]
    pools[:, 1, 0], pools[:, 1, 1] = b.k, b.v
    wide = torch.full((b.total, 12, 64), NAN, dtype=t, device="cuda")
    wide[:, 3:7] = b.q
    out = torch.full((b.total, 6, 64), 7.0, dtype=t, device="cuda")
    tab = torch.full((2, 20), -1, dtype=torch.int32, device="cuda")
    tab[:, :9] = b.table
    kv = paged.PagedKv(pools[:, 1, 0], pools[:, 1, 1])
    kv.attention(wide[:, 3:7], tab[:, :9], b.row_start, b.kv_len, max_rows=12, out=out[:, 1:5])
    b.check(out[:, 1:5])
    assert bool((out[:, 0] == 7.0).all()) and bool((out[:, 5] == 7.0).all())


@pytest.mark.parametrize("t", TYPES)
def test_strides_that_are_never_stepped_over_do_not_count(t):
    """A single row of Q, K, V and the result in rows of odd length, a pool with one head, one page and pages of one row."""
    for page, hkv in ((16, 1), (1, 2)):
        b = Batch([1], [1 if page == 1 else 9], 4, hkv, 64, t, page, "head", spare=0)
        one = lambda x: torch.empty(x.shape[1] * 64 + 3, dtype=t, device="cuda")[:x.shape[1] * 64].view(1, -1, 64).as_strided(x.shape, (x.shape[1] * 64 + 3, 64, 1))
        q, out, k = one(b.q), one(b.q), one(b.q[:, :hkv])
        q.copy_(b.q)
        odd = lambda x: x.as_strided(x.shape, [s if n > 1 else 4097 for n, s in zip(x.shape, x.stride())])
        kv = paged.PagedKv(odd(b.k), b.v)
        kv.attention(q, b.table, b.row_start, b.kv_len, max_rows=1, out=out)
        b.check(out)
        k.copy_(torch.randn(1, hkv, 64))
        kv.append(k, k, b.table, b.row_start, b.kv_len)
        place = (int(b.table_h[0, (b.lens[0] - 1) // page]), (b.lens[0] - 1) % page)
        for pool in (b.k, b.v):
            assert torch.equal(b.cell(pool, *place), k[0].to(PAGE[t]))


def test_a_long_cache_is_addressed_past_32_bits():
    """A pool whose last pages lie beyond 2^32 bytes and 2^31 elements: the same keys there and at its start."""
    page, hkv, d = 64, 8, 128
    n_pages = (1 << 32) // (page * hkv * d) + 8  # 2^32 elements and a little, 8 GiB each
    k = torch.empty(n_pages, hkv, page, d, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    b = Batch([1, 30], [200, 100], 16, hkv, d, F16, page, "head", spare=0)
    far = torch.arange(b.n_pages, device="cuda") + (n_pages - b.n_pages)
    k[far], v[far] = b.k, b.v
    kv = paged.PagedKv(k, v)
    high = torch.where(b.table >= 0, b.table + (n_pages - b.n_pages), b.table)
    out = kv.attention(b.q, high, b.row_start, b.kv_len, max_rows=30)
    b.check(out)
    new = torch.randn(b.total, hkv, d).half().cuda()
    kv.append(new, new, high, b.row_start, b.kv_len)
    last = int(high[0, (200 - 1) // page])
    assert torch.equal(v[last, :, (200 - 1) % page], new[0])


def test_results_do_not_change_between_runs():
    b = Batch([1] * 9, [700, 3, 900, 64, 65, 1, 512, 333, 128], 8, 2, 128, BF16, 16, "head")
    first = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1)
    for _ in range(3):
        assert torch.equal(PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1), first)
    b = Batch([70, 1, 300], [700, 33, 300], 8, 2, 128, BF16, 16, "head")
    first = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=300)
    for _ in range(3):
        assert torch.equal(PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=300), first)


# ---- batches that give a CTA many tiles, or many cells ------------------------------------------------------------------------


def run_device_batch(b, window=0, scale=None, **kw):
    out = torch.full((b.total, b.hq, b.d), 7.0, dtype=b.t, device="cuda")
    lse = torch.full((b.total, b.hq), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=max(b.rows), window=window, scale=scale, out=out, lse=lse, status=status)
    assert int(status) == 0
    b.check(out, lse, window, scale, **kw)
    return out, lse


def processors():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (4, 1, 128), (3, 1, 96)])
@pytest.mark.parametrize("window", [0, 40])
def test_many_short_cells_one_behind_the_other(t, hq, hkv, d, window):
    """Cells of one to three tiles, dozens in a CTA: blocks that both streams share (one of them often without a tile), blocks
    of their own, and rows that see nothing of a stream's share, in every order."""
    rng = np.random.default_rng(d + window)
    n_seqs = 600
    rows = [int(x) for x in rng.choice([1, 3, 20, 31, 40, 65, 100, 150], n_seqs)]
    lens = [r + int(x) for r, x in zip(rows, rng.choice([0, 0, 5, 27, 100, 128, 260], n_seqs))]
    pieces = plan_tc(rows, lens, hq // hkv, hkv, window, processors())
    assert max(np.bincount([p[0] for p in pieces])) >= 5
    assert {1, 2} <= {p[2] for p in pieces if p[1] <= 128} and {1, 2} <= {p[2] for p in pieces if p[1] > 128}
    b = DeviceBatch(rows, lens, hq, hkv, d, t, 16, "head", seed=d)
    first = run_device_batch(b, window)
    for _ in range(5):
        out, lse = torch.empty_like(first[0]), torch.empty_like(first[1])
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=max(b.rows), window=window, out=out, lse=lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def growing(q, k, v):
    """Scores that climb along the keys, by several of the lazy steps, for the even rows; that fall for the odd ones; and that
    swing for every third one."""
    rows, n = q.shape[0], k.shape[0]
    x = torch.linspace(0, 1, n, device="cuda")[:, None, None]
    axis = torch.zeros(q.shape[-1], device="cuda")
    swing, climb = axis.clone(), axis.clone()
    climb[0::2], swing[1::2] = 1.0, 1.0
    k = 0.3 * k + 6.0 * (x * climb + torch.sin(25 * x) * swing)
    r = torch.arange(rows, device="cuda")[:, None, None]
    q = 0.3 * q + torch.where(r % 3 == 2, 1.0, 0.0) * swing + torch.where(r % 2 == 0, 1.0, -1.0) * torch.where(r % 3 == 2, 0.0, 1.0) * climb
    return q, k, v


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d,page,layout", [(64, 16, "token"), (128, 64, "head"), (128, 8, "head"), (40, 256, "token")])
@pytest.mark.parametrize("shape", [None, growing])
@pytest.mark.parametrize("window", [0, 1500])
def test_runs_of_many_tiles_on_the_tensor_memory_kernel(t, d, page, layout, shape, window):
    """Batches that give a CTA's streams many tiles of a cell, of blocks that both share (two sequences of few rows) and of
    blocks of their own, cells that two, three and more CTAs have a part of, and several cells in a CTA."""
    rows, lens = [300, 40, 1, 129, 33, 260, 0, 64], [4100, 12000, 3000, 1500, 9001, 2049, 500, 6000]
    if window:
        rows, lens = 3 * rows, 3 * lens
    hq, hkv = 8, 4
    pieces = plan_tc(rows, lens, hq // hkv, hkv, window, processors())
    own, shared = [p for p in pieces if p[1] > 128], [p for p in pieces if p[1] <= 128]
    assert max(p[2] for p in own) >= 6 and max(p[2] for p in shared) >= 8
    parts = np.bincount([p[4] for p in pieces])
    assert {1, 2} <= set(parts) and (window or max(parts) >= 4)
    assert any(p[2] < p[3] for p in own) and any(p[2] < p[3] for p in shared)
    assert max(np.bincount([p[0] for p in pieces])) >= 2
    b = DeviceBatch(rows, lens, hq, hkv, d, t, page, layout, seed=d + page, shape=shape)
    first = run_device_batch(b, window)
    for _ in range(3):
        out, lse = torch.empty_like(first[0]), torch.empty_like(first[1])
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=max(b.rows), window=window, out=out, lse=lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def halves_alike(q, k, v):
    half = v.shape[-1] // 2
    return q, k, torch.cat((v[..., :half], v[..., :half]), -1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,parts", [([4000, 2300, 9001], {5, 8, 18}), ([1500, 700] * 12, {1, 2})])
def test_both_halves_of_the_channels_are_weighed_alike(t, d, lens, parts):
    """Blocks that both streams share are finished by two warpgroups, half of the channels each, and joined by whichever CTA
    comes last: values whose halves are the same give halves that are the same, to the bit - a sum that the two held
    differently would also make the bits of a result depend on who came last."""
    rows = ([33, 40, 50] * 8)[:len(lens)]
    pieces = plan_tc(rows, lens, 2, 4, 0, processors())
    assert all(p[1] <= 128 for p in pieces)
    if processors() == 148:
        assert parts <= set(np.bincount([p[4] for p in pieces]))
    b = DeviceBatch(rows, lens, 8, 4, d, t, 16, "head", seed=d, shape=halves_alike)
    first = run_device_batch(b)
    assert torch.equal(first[0][..., :d // 2], first[0][..., d // 2:])
    for _ in range(20):
        out, lse = torch.empty_like(first[0]), torch.empty_like(first[1])
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=max(b.rows), out=out, lse=lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_whole_cells_of_many_tiles(t, d):
    """More cells than CTAs, each of 20 tiles: nothing is joined, every stream runs its cells' tiles through."""
    rows, lens = [160] * 40, [2560 - 37 * i for i in range(40)]
    pieces = plan_tc(rows, lens, 2, 4, 0, processors())
    assert max(p[2] for p in pieces) >= 16 and any(p[2] == p[3] >= 10 for p in pieces if p[1] > 128) and any(p[2] == p[3] >= 10 for p in pieces if p[1] <= 128)
    run_device_batch(DeviceBatch(rows, lens, 8, 4, d, t, 32, "head", seed=d, shape=growing))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("shape", [None, growing])
@pytest.mark.parametrize("window", [0, 2100])
def test_runs_of_many_tiles_on_the_streaming_kernel(t, d, rows, shape, window):
    """The same for its narrow and its wide block: 8 and 24 pairs, dozens of tiles of a cell in a CTA."""
    hq, hkv = 64, 8
    lens = [4000 + 311 * i for i in range(16)]
    narrow = 8 if t is F32 else 16
    block = 2 * narrow if rows * hq // hkv > narrow and d <= 128 else narrow
    pieces = plan_stream([rows] * 16, lens, hq // hkv, hkv, window, block, (2 if d <= 128 else 1) * processors())
    assert max(p[1] for p in pieces) >= 14 and any(p[1] < p[2] for p in pieces)
    run_device_batch(DeviceBatch([rows] * 16, lens, hq, hkv, d, t, 16, "token", seed=d, shape=shape), window)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("below", [9.3, 13.2, 16.4, 18.7, 21.55])
def test_one_key_far_above_many_small_ones(t, d, rows, below):
    """A key whose weight is 2^below times that of each of some thousand others, which all count the same way: a step of the
    weights' type, times their number, must not show.  Half pages keep a weight to 2^-25 in a scale where the largest is 2^7 at
    least, 2^-32 of it; bf16 has no such step."""
    def sink(q, k, v):
        q, k, v = torch.zeros_like(q), torch.zeros_like(k), torch.ones_like(v)
        # the first key's score above the others': 4 k times 2^-x, a scale of ln(2) and a common factor
        q[..., 0], k[..., 0] = 4.0, -below / 4.0
        k[0, :, 0], v[0] = 0.0, 0.0
        return q, k, v

    b = DeviceBatch([rows] * 2, [8192, 3001], 4, 2, d, t, 16, "head", shape=sink)
    run_device_batch(b, scale=math.log(2.0), step=0.0 if t is BF16 else 2.0 ** -32)


@pytest.fixture
def short_waits():
    yield paged.wait_limit
    torch.cuda.synchronize()
    paged.wait_limit(0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_a_wait_that_runs_out_shows(short_waits, t, d):
    """With bounds far below what a tile takes: rows come out as they would have or as NaN, never as something else, the
    status says so, and the workspace serves the next call."""
    rows, lens = [300, 40, 1, 129, 33, 260, 0, 64] * 2, [1100, 4000, 300, 500, 2001, 1049, 500, 900] * 2
    b = DeviceBatch(rows, lens, 8, 4, d, t, 16, "head", seed=d)
    pieces = plan_tc(rows, lens, 2, 4, 0, processors())
    parts = np.bincount([p[4] for p in pieces])
    assert {1, 2} <= set(parts) and max(parts) >= 3 and max(np.bincount([p[0] for p in pieces])) >= 2
    ws, status = paged.attention_workspace("cuda:0"), torch.zeros(1, dtype=torch.int32, device="cuda")
    n_tickets = 4 * 2 * processors()

    def run():
        out, lse = torch.full((b.total, 8, d), 7.0, dtype=t, device="cuda"), torch.full((b.total, 8), 7.0, device="cuda")
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=300, out=out, lse=lse, workspace=ws, status=status)
        torch.cuda.synchronize()
        assert bool((ws[:n_tickets] == 0).all())
        return out, lse

    want = run()
    assert int(status) == 0
    lost = []
    for limit in (1, 3, 8):
        short_waits(limit)
        status.zero_()
        out, lse = run()
        gone = torch.isnan(lse)
        lost.append(int(gone.sum()))
        assert int(status) in ((16,) if lost[-1] else (0, 16))
        assert bool(torch.isnan(out[gone]).all())
        assert torch.equal(out[~gone], want[0][~gone]) and torch.equal(lse[~gone], want[1][~gone])
    assert lost[0] > 0
    short_waits(0)
    status.zero_()
    again = run()
    assert int(status) == 0 and torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


# ---- streams, graphs, workspaces ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 40])
def test_another_stream_and_one_given_by_number(rows):
    b = Batch([rows] * 3, [rows + 5, 200, 77], 4, 2, 64, F16, 16, "head")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows)
    out2 = torch.empty_like(out)
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows, out=out2, stream=s.cuda_stream)
    s.synchronize()
    b.check(out)
    assert torch.equal(out, out2)


def calls_with_a_result_of_their_own():
    f, fd, _ = table(64)
    x, pos = torch.randn(48, 4, 64, device="cuda"), torch.arange(48, dtype=torch.int32, device="cuda")
    b = Batch([16] * 3, [21, 200, 77], 4, 2, 64, F32, 16, "head")
    k = torch.randn(48, 2, 64, device="cuda")
    kv, batch = PagedOf(b), (b.table, b.row_start, b.kv_len)
    return {"rope": lambda **kw: paged.rope_apply(x, pos, fd, **kw),
            "append": lambda **kw: kv.append(k, k, *batch, q=x, inv_freq=fd, **kw),
            "attention": lambda **kw: kv.attention(x, *batch, max_rows=1, **kw)}


@pytest.mark.parametrize("name", ["rope", "append", "attention"])
def test_a_result_that_another_stream_writes_is_that_streams_memory(name):
    """A block that work queued on the current stream still reads, freed behind that work, is not what a call on another
    stream writes its result to - nor is the result's block handed out on the current stream while that one writes."""
    call = calls_with_a_result_of_their_own()[name]
    want = call()  # (also the first call of its kind)
    s = torch.cuda.Stream()
    call(stream=s.cuda_stream)
    torch.cuda.synchronize()
    held = torch.full_like(want, 5.0)
    read = torch.empty_like(held)
    torch.cuda._sleep(1 << 26)  # some 30 ms before the block is read
    read.copy_(held)
    at = held.data_ptr()
    del held
    got = call(stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert bool((read == 5.0).all()), "a block that was still being read was written"
    assert torch.equal(got, want) and got.data_ptr() != at
    at = got.data_ptr()
    del got
    assert torch.empty_like(want).data_ptr() != at  # it went back to the other stream
    # the same stream by number: as without it
    assert torch.equal(call(stream=torch.cuda.current_stream().cuda_stream), want)


def test_two_streams_at_once():
    b = [Batch([1] * 4, [900, 40, 333, 64], 8, 2, 128, F16, 16, "head", seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in b]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for x, s in zip(b, streams):
            with torch.cuda.stream(s):
                outs.append(PagedOf(x).attention(x.q, x.table, x.row_start, x.kv_len, max_rows=1))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, outs[i % 2])
    b[0].check(outs[0])
    b[1].check(outs[1])


def test_a_captured_call_needs_a_workspace_of_its_own():
    b = Batch([1], [40], 4, 2, 64, F16, 16, "head")
    out = torch.empty_like(b.q)
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(CudaComputeError) as e:
            PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, out=out)
    assert "workspace" in e.value.msg


def test_a_stream_given_by_number_that_is_being_captured_needs_a_workspace_too():
    b = Batch([1], [40], 4, 2, 64, F16, 16, "head")
    out = torch.empty_like(b.q)
    captured, current = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (captured, current):  # each has a workspace of the module's
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, out=out, stream=s.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=captured):
        with torch.cuda.stream(current), pytest.raises(CudaComputeError) as e:
            PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, out=out, stream=captured.cuda_stream)
    assert "workspace" in e.value.msg


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("captured", [False, True])
def test_tables_and_lengths_that_the_kernel_before_wrote(rows, captured):
    """The kernels take their places while the one before them still runs: what it wrote last is what they read."""
    b = Batch([rows] * 3, [700, 260, 513], 8, 2, 64, F16, 16, "head")
    kv, ws = PagedOf(b), paged.attention_workspace("cuda:0")
    other = b.table.flip(0).contiguous()  # the sequences in the opposite order
    lens = [b.kv_len.clone(), b.kv_len.flip(0).contiguous()]
    tables = [b.table.clone(), other]
    want = [kv.attention(b.q, tables[i], b.row_start, lens[i], max_rows=rows, workspace=ws) for i in (0, 1)]
    outs = [torch.empty_like(b.q) for _ in range(2)]
    turn = torch.zeros(1, dtype=torch.int64, device="cuda")
    both, both_lens = torch.stack(tables), torch.stack(lens)

    def steps():
        for _ in range(10):
            for out in outs:
                b.table.copy_(both.index_select(0, turn)[0] + 0 * b.table)  # (reads what it replaces)
                b.kv_len.copy_(both_lens.index_select(0, turn)[0])
                turn.sub_(1).neg_()
                kv.attention(b.q, b.table, b.row_start, b.kv_len, max_rows=rows, out=out, workspace=ws)

    torch.cuda.synchronize()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            steps()
    for _ in range(10):
        for out in outs:
            out.zero_()
        g.replay() if captured else steps()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_the_per_thread_default_stream_shares_nothing_of_the_modules():
    """Its handle is one number for the streams of all threads: neither a workspace nor the allocator may go by it."""
    b = Batch([1, 1], [400, 90], 4, 2, 64, F16, 16, "head")
    args, per_thread = (b.q, b.table, b.row_start, b.kv_len), 2
    ws = [paged.attention_workspace("cuda:0") for _ in range(4)]
    outs = [torch.empty_like(b.q) for _ in ws]
    with pytest.raises(CudaComputeError) as e:
        PagedOf(b).attention(*args, max_rows=1, out=outs[0], stream=per_thread)
    assert "workspace" in e.value.msg
    for call in (lambda: PagedOf(b).attention(*args, max_rows=1, workspace=ws[0], stream=per_thread),
                 lambda: paged.rope_apply(b.q, torch.zeros(2, dtype=torch.int32, device="cuda"), table(64)[1], stream=per_thread),
                 lambda: PagedOf(b).append(b.q[:, :2], b.q[:, 2:], b.table, b.row_start, b.kv_len, q=b.q, stream=per_thread)):
        with pytest.raises(CudaComputeError) as e:
            call()
        assert "memory" in e.value.msg
    torch.cuda.synchronize()

    def thread(i):
        for _ in range(20):
            PagedOf(b).attention(*args, max_rows=1, out=outs[i], workspace=ws[i], stream=per_thread)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(ws))]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    torch.cuda.synchronize()
    for o in outs:
        b.check(o)


def test_a_workspace_is_not_made_inside_a_capture():
    b = Batch([1], [40], 4, 2, 64, F16, 16, "head")
    out = torch.empty_like(b.q)
    fresh = torch.cuda.Stream()  # (a stream whose workspace is not there yet)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    paged._workspaces.pop((0, fresh.cuda_stream), None)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.add_(1)
        for call in (lambda: paged.attention_workspace("cuda:0"),
                     lambda: PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, out=out, stream=fresh.cuda_stream)):
            with pytest.raises(CudaComputeError) as e:
                call()
            assert "captured" in e.value.msg
    g.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())  # the capture went on


@pytest.mark.parametrize("name", ["rope", "append", "attention"])
def test_autograd_is_not_passed_by_in_silence(name):
    """A tensor that requires a gradient is refused rather than detached; one that autograd has saved counts as changed."""
    f, fd, _ = table(64)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    b = Batch([4], [9], 2, 2, 64, F32, 8, "head")
    kv, batch = PagedOf(b), (b.table, b.row_start, b.kv_len)
    x, k = torch.randn(4, 2, 64, device="cuda"), torch.randn(4, 2, 64, device="cuda")
    call = {"rope": lambda x, out: paged.rope_apply(x, pos, fd, out=out),
            "append": lambda x, out: kv.append(k, k, *batch, q=x, q_out=out, inv_freq=fd),
            "attention": lambda x, out: kv.attention(x, *batch, max_rows=4, out=out)}[name]
    leaf = x.clone().requires_grad_()
    for kw in (dict(x=leaf, out=torch.empty_like(x)), dict(x=leaf * 2, out=torch.empty_like(x)), dict(x=x, out=leaf)):
        with pytest.raises(CudaComputeError) as e:
            call(**kw)
        assert "gradient" in e.value.msg
    with torch.no_grad():
        want = call(leaf, torch.empty_like(x)).clone()
    assert not want.requires_grad and torch.equal(want, call(x, torch.empty_like(x)))
    with torch.inference_mode():
        assert torch.equal(want, call(x, torch.empty_like(x)))
    w = torch.ones(4, 2, 64, device="cuda", requires_grad=True)
    out = x.clone()
    y = (w * out).sum()  # saves out
    call(x, out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rows_of_another_number_of_dimensions_are_refused():
    b = Batch([1], [40], 4, 2, 64, F16, 16, "head")
    for k in (b.q[0, 0, 0], b.q[0], b.q[None]):
        with pytest.raises(CudaComputeError):
            PagedOf(b).append(k, k, b.table, b.row_start, b.kv_len)
        with pytest.raises(CudaComputeError):
            PagedOf(b).attention(k, b.table, b.row_start, b.kv_len, max_rows=1)


def test_the_modules_workspaces_are_given_up():
    b = Batch([1], [400], 4, 2, 64, F16, 16, "head")
    PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1)
    assert paged._workspaces
    paged.release_workspaces()
    assert not paged._workspaces
    b.check(PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1))
    assert len(paged._workspaces) == 1


def test_a_workspace_that_is_too_small_is_refused():
    b = Batch([1], [40], 4, 2, 64, F16, 16, "head")
    ws = paged.attention_workspace("cuda:0")
    with pytest.raises(CudaComputeError) as e:
        PagedOf(b).attention(b.q, b.table, b.row_start, b.kv_len, max_rows=1, workspace=ws[:-256])
    assert e.value.code == _lib.ERR_CAPACITY


@pytest.mark.parametrize("t", TYPES)
def test_the_operators_together_in_a_replayed_step(t):
    """A prompt's chunk, then decode steps that a graph replays: each step rotates and stores its token and attends, the
    lengths moving on the device.  Against the same run in 64 bits on the values that the pages hold."""
    hq, hkv, d, page, n0, steps = 4, 2, 64, 16, 45, 5
    f, fd, m = table(d, scaling="bands", factor=8.0, original_context=256.0, low=1.0, high=4.0)
    seqs = 3
    lens = [n0, 17, 1]
    width = 6
    g = torch.Generator().manual_seed(3)
    pt = PAGE[t]
    k_pool, v_pool = (torch.full((seqs * width, page, hkv, d), NAN, dtype=pt, device="cuda") for _ in range(2))
    tab = torch.randperm(seqs * width, generator=g).to(torch.int32).view(seqs, width).cuda()
    kv = paged.PagedKv(k_pool, v_pool, layout="token")
    ws = paged.attention_workspace("cuda:0")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def host_rows(s, n):
        ids = tab[s].cpu().long()
        at = torch.arange(n)
        return (p.cpu()[ids[at // page], at % page].double() for p in (k_pool, v_pool))

    def check(qr, out, rows, lens):
        b = Batch.__new__(Batch)
        b.rows, b.lens, b.hq, b.hkv, b.d, b.t = rows, lens, hq, hkv, d, t
        b.starts = np.cumsum([0] + rows).tolist()
        b.q_h = qr.cpu()
        pairs = [tuple(host_rows(s, n)) for s, n in enumerate(lens)]
        b.keys, b.values = [p[0] for p in pairs], [p[1] for p in pairs]
        b.check(out)

    def layer(qkv, row_start, kv_len, q_rot, out, max_rows):
        kv.append(qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], tab, row_start, kv_len, q=qkv[:, :hq], q_out=q_rot, inv_freq=fd, pairing=1,
                  magnitude=m, status=status)
        kv.attention(q_rot, tab, row_start, kv_len, max_rows=max_rows, out=out, workspace=ws, status=status)

    total = sum(lens)
    qkv = torch.randn(total, hq + 2 * hkv, d, generator=g).to(t).cuda()
    q_rot, out = (torch.empty(total, hq, d, dtype=t, device="cuda") for _ in range(2))
    starts = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
    layer(qkv, starts, torch.tensor(lens, dtype=torch.int32, device="cuda"), q_rot, out, max(lens))
    check(q_rot, out, lens, lens)
    for s, n in enumerate(lens):  # what the prompt left in the pages
        k_row, _ = host_rows(s, n)
        x = qkv[starts[s]:starts[s] + n, hq:hq + hkv].cpu()
        extra, _ = rotation_bound(x, f, 1, m, pt)
        within(k_row, rotate(x, torch.arange(n), f, 1, m), extra, pt)

    kv_len = torch.tensor([n + 1 for n in lens], dtype=torch.int32, device="cuda")
    one = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    step_in = torch.zeros(seqs, hq + 2 * hkv, d, dtype=t, device="cuda")
    q1, out1 = (torch.empty(seqs, hq, d, dtype=t, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(step_in, one, kv_len, q1, out1, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(step_in, one, kv_len, q1, out1, 1)
        kv_len.add_(1)
    for i in range(steps):
        step_in.copy_(torch.randn(seqs, hq + 2 * hkv, d, generator=g).to(t))
        graph.replay()
        check(q1, out1, [1] * seqs, [n + 1 + i for n in lens])
        want = rotate(step_in[:, :hq].cpu(), [n + i for n in lens], f, 1, m)
        extra, _ = rotation_bound(step_in[:, :hq].cpu(), f, 1, m, t)
        within(q1, want, extra, t)
    assert int(status) == 0


def test_pool_objects_refuse_what_they_cannot_describe():
    k = torch.zeros(4, 2, 16, 64, dtype=F16, device="cuda")
    for bad in (lambda: paged.PagedKv(k, k[:3]), lambda: paged.PagedKv(k.float(), k.float()), lambda: paged.PagedKv(k.cpu(), k.cpu()),
                lambda: paged.PagedKv(k, k, layout="rows"), lambda: paged.PagedKv(k[..., ::2], k[..., ::2]), lambda: paged.PagedKv(k[0], k[0]),
                lambda: paged.PagedKv(k, k.bfloat16())):
        with pytest.raises(CudaComputeError):
            bad()
    kv = paged.PagedKv(k, k.clone())
    i32 = dict(dtype=torch.int32, device="cuda")
    q, tab, st, ln = torch.zeros(2, 4, 64, dtype=F16, device="cuda"), torch.zeros(2, 3, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32)
    for kw in (dict(q=q.bfloat16()), dict(q=q[..., :32]), dict(q=q.float().double()), dict(tab=tab.long()), dict(tab=tab[:1]), dict(st=st[:2]), dict(ln=ln.cpu()),
               dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(out=q[:1]), dict(lse=torch.zeros(2, 3, device="cuda")), dict(window=-1), dict(window=2 ** 32), dict(scale=1e300),
               dict(status=torch.zeros(1, device="cuda")), dict(workspace=torch.zeros(10, device="cuda")), dict(q=torch.zeros(2, 3, 64, dtype=F16, device="cuda"))):
        a = dict(q=q, tab=tab, st=st, ln=ln)
        a.update(kw)
        with pytest.raises(CudaComputeError):
            kv.attention(a.pop("q"), a.pop("tab"), a.pop("st"), a.pop("ln"), max_rows=1, **a)
    assert kv.attention(q[:0], tab, st, ln, max_rows=0).shape == (0, 4, 64)
    with pytest.raises(CudaComputeError):  # heads that are not contiguous, rows or not
        kv.append(k[0, :, :0].transpose(0, 1), k[0, :, :0].transpose(0, 1), tab, st, ln)
    assert kv.append(q[:0, :2], q[:0, 2:], tab, st, ln) is None
