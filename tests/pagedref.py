"""The paged operators from their definitions, in 64 bits on the host, one row and head at a time, and how far a device
result may be from them.

Rounding one value to a type t is off by at most u = eps(t) / 2 of it (bf16 2^-8, f16 2^-11, f32 2^-24)."""
import math

import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
PAGE = {torch.float32: torch.float16, torch.float16: torch.float16, torch.bfloat16: torch.bfloat16}


def rotate(x, positions, inv_freq, pairing, magnitude=1.0, inverse=False):
    """x [rows][heads][D] f64 tensor, as complex pairs times magnitude * exp(+-i angle)."""
    x = x.double().clone()
    n = len(inv_freq)
    a = torch.arange(n) * (2 if pairing == 0 else 1)
    b = a + (1 if pairing == 0 else n)
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None] * torch.as_tensor(np.asarray(inv_freq), dtype=torch.float64)
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)[:, None]
    x[..., a], x[..., b] = z.real, z.imag
    return x


def rotation_bound(x, inv_freq, pairing, magnitude, t):
    """|x_a cos - x_b sin| in f32: sine and cosine are within 2^-24 * pi (the reduced angle's rounding, at most half a
    turn of half turns) + 2 * 2^-24 (sincospif, 1 ulp-grade, and the product with the magnitude) of the exact ones; two products and a sum
    round 3 times more: 9 * 2^-24 of |x_a| + |x_b| covers it.  Then one rounding to t."""
    n = len(inv_freq)
    a = torch.arange(n) * (2 if pairing == 0 else 1)
    b = a + (1 if pairing == 0 else n)
    size = x.double().abs().clone()
    both = (x.double()[..., a].abs() + x.double()[..., b].abs()) * abs(magnitude)
    size[..., a], size[..., b] = both, both
    extra = torch.zeros(x.shape[-1], dtype=torch.float64)
    extra[a], extra[b] = 9 * 2.0 ** -24, 9 * 2.0 ** -24
    return size * extra, size


def within(got, want, err, t):
    """|got - want| <= err + one rounding to t (and t's subnormal step)."""
    got, want = got.double().cpu(), want.double()
    tiny = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[t]
    off = (got - want).abs()
    bound = err * (1 + U[t]) + U[t] * want.abs() + tiny
    bad = off > bound
    assert not bool(bad.any()) and bool(torch.isfinite(got).all()), (
        f"{int(bad.sum())} of {bad.numel()} values off, worst {float((off - bound).max()):.3e} over a bound of "
        f"{float(bound.reshape(-1)[int((off - bound).argmax())]):.3e}")


def attend(q, keys, values, pos0, scale, window):
    """One sequence: q [rows][Hq][D], keys / values [n][Hkv][D] (f64): (out, lse, mean, slack).  mean = sum of weight *
    |value|: what the rounding of weights and sums is proportional to; slack = the f32 score's error bound."""
    rows, hq, d = q.shape
    n, hkv, _ = keys.shape
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    mean, slack = torch.zeros_like(out), torch.zeros(rows, hq, dtype=torch.float64)
    for r in range(rows):
        p = pos0 + r
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        if p < 0 or hi <= lo:
            continue
        for h in range(hq):
            k, v = keys[lo:hi, h // (hq // hkv)], values[lo:hi, h // (hq // hkv)]
            s = k @ q[r, h] * scale
            top = s.max()
            w = torch.exp(s - top)
            lse[r, h] = top + w.sum().log()
            out[r, h] = (w / w.sum()) @ v
            mean[r, h] = (w / w.sum()) @ v.abs()
            slack[r, h] = (k.abs() @ q[r, h].abs()).max() * abs(scale)
    return out, lse, mean, slack


def attend_bound(mean, slack, n, d, t):
    """How far an output may be, before its own rounding: scores are sums of d products in f32 (and, for f32 rows, of
    products good to 2^-21 of their size), so a weight is off by the factor 1 +- 2 e with e = (d + 16) 2^-24 * slack; the
    weight itself is rounded to the pages' type for 16-bit rows (u) and to two halfs for f32 rows (2^-21, and 2^-23 of
    the exponential); sums over n keys run in f32 in steps of 16 keys; joins and the quotient add a few roundings."""
    weight = 2.0 ** -21 if t is torch.float32 else U[t]
    e = 2 * ((d + 16) * 2.0 ** -24 + (2.0 ** -21 if t is torch.float32 else 0.0)) * slack
    return mean * (weight + (n / 16 + 64) * 2.0 ** -24 + e[..., None])


class Batch:
    """A ragged batch on the device with its host copies: ``rows`` and ``lens`` per sequence, pages scattered over the pool
    whose unused rows hold NaN."""

    def __init__(self, rows, lens, hq, hkv, d, t, page, layout, seed=0, extra_rows=0, spare=2, width=None, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.hq, self.hkv, self.d, self.t, self.page, self.layout = rows, lens, hq, hkv, d, t, page, layout
        pt = PAGE[t]
        held = [-(-n // page) for n in lens]
        self.n_pages = sum(held) + spare
        self.width = max(1, max(held)) if width is None else width
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((len(rows), self.width), -1, dtype=torch.int32)
        i = 0
        for s, n in enumerate(held):
            table[s, :n] = torch.tensor(order[i:i + n], dtype=torch.int32)
            i += n
        self.table_h = table
        self.keys = [torch.randn(n, hkv, d, generator=g).to(pt) for n in lens]
        self.values = [torch.randn(n, hkv, d, generator=g).to(pt) for n in lens]
        shape = (self.n_pages, hkv, page, d) if layout == "head" else (self.n_pages, page, hkv, d)
        self.k_h, self.v_h = (torch.full(shape, math.nan, dtype=pt) for _ in range(2))
        for s, n in enumerate(lens):
            for p in range(n):
                for pool, src in ((self.k_h, self.keys), (self.v_h, self.values)):
                    self.cell(pool, int(table[s, p // page]), p % page).copy_(src[s][p])
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        self.total = starts[-1] + extra_rows
        self.starts = starts
        self.q_h = torch.randn(self.total, hq, d, generator=g).to(t)
        self.k = self.k_h.to(device)
        self.v = self.v_h.to(device)
        self.table = table.to(device)
        self.row_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=device)
        self.q = self.q_h.to(device)

    def cell(self, pool, page, row):
        """[kv_heads][D] view of one row of one page."""
        return pool[page, :, row] if self.layout == "head" else pool[page, row]

    def check(self, out, lse=None, scale=None, window=0, only=None):
        scale = 1.0 / math.sqrt(self.d) if scale is None else scale
        scale = float(np.float32(scale))
        for s, (r, n) in enumerate(zip(self.rows, self.lens)):
            if r == 0 or (only is not None and s not in only):
                continue
            lo = self.starts[s]
            want, want_lse, mean, slack = attend(self.q_h[lo:lo + r].double(), self.keys[s].double(), self.values[s].double(),
                                                 n - r, scale, window)
            err = attend_bound(mean, slack, n, self.d, self.t)
            within(out[lo:lo + r], want, err, self.t)
            if lse is not None:
                got = lse[lo:lo + r].double().cpu()
                seen = torch.isfinite(want_lse)
                assert torch.equal(torch.isfinite(got), seen) and bool((got[~seen] == -math.inf).all())
                # the score's error, the sum's, and log2 and its product in f32
                tol = (self.d + 16) * 2.0 ** -24 * slack + 2.0 ** -20 * slack + (n / 16 + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * want_lse.abs()
                assert bool(((got - want_lse).abs()[seen] <= tol[seen]).all()), float((got - want_lse).abs()[seen].max())


# ---- the same for batches of some thousand keys, on the device ----------------------------------------------------------

def attend_many(q, keys, values, pos0, scale, window):
    """``attend`` with all rows and heads of a sequence at once, on the tensors' own device."""
    rows, hq, d = q.shape
    n, hkv, _ = keys.shape
    k, v = (x.double().transpose(0, 1).repeat_interleave(hq // hkv, 0) for x in (keys, values))  # [Hq][n][D]
    qh = q.double().transpose(0, 1)
    p = torch.arange(pos0, pos0 + rows, device=q.device)[:, None]
    key = torch.arange(n, device=q.device)
    seen = (key <= p) & (key > p - window) if window else key <= p
    s = (qh @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    lse = (top + total.log()).squeeze(-1)
    slack = (qh.abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(-1) * abs(scale)
    return (w @ v).transpose(0, 1), lse.transpose(0, 1), (w @ v.abs()).transpose(0, 1), slack.transpose(0, 1)


class DeviceBatch:
    """A ragged batch made on the device, pages scattered over a pool whose unused rows hold NaN.  ``shape``: what to do with
    (q, keys, values) of a sequence before they are stored."""

    def __init__(self, rows, lens, hq, hkv, d, t, page, layout, seed=0, shape=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.lens, self.hq, self.hkv, self.d, self.t, self.page, self.layout = rows, lens, hq, hkv, d, t, page, layout
        pt, i32 = PAGE[t], dict(dtype=torch.int32, device="cuda")
        held = [-(-n // page) for n in lens]
        self.n_pages = sum(held) + 2
        order = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(rows), max(1, max(held))), -1, **i32)
        self.starts = np.cumsum([0] + rows).tolist()
        self.total = self.starts[-1]
        self.k, self.v = (torch.full((self.n_pages, page, hkv, d), math.nan, dtype=pt, device="cuda") for _ in range(2))
        self.q = torch.empty(self.total, hq, d, dtype=t, device="cuda")
        self.keys, self.values = [], []
        for s, (r, n) in enumerate(zip(rows, lens)):
            at = sum(held[:s])
            self.table[s, :held[s]] = order[at:at + held[s]]
            q, k, v = (torch.randn(m, h, d, generator=g, device="cuda") for m, h in ((r, hq), (n, hkv), (n, hkv)))
            if shape is not None:
                q, k, v = shape(q, k, v)
            self.q[self.starts[s]:self.starts[s] + r] = q.to(t)
            self.keys.append(k.to(pt))
            self.values.append(v.to(pt))
            p = torch.arange(n, device="cuda")
            place = (self.table[s].long()[p // page], p % page)
            self.k[place], self.v[place] = self.keys[s], self.values[s]
        if layout == "head":
            self.k, self.v = (x.transpose(1, 2).contiguous() for x in (self.k, self.v))
        self.row_start = torch.tensor(self.starts, **i32)
        self.kv_len = torch.tensor(lens, **i32)

    def check(self, out, lse, window=0, scale=None, step=0.0):
        """``step``: what a weight may be off by beyond its relative rounding, as a share of the row's largest."""
        scale = float(np.float32(1.0 / math.sqrt(self.d) if scale is None else scale))
        for s, (r, n) in enumerate(zip(self.rows, self.lens)):
            if r == 0:
                continue
            lo = self.starts[s]
            want, want_lse, mean, slack = (x.cpu() for x in attend_many(self.q[lo:lo + r], self.keys[s], self.values[s], n - r, scale, window))
            small = step * float(self.values[s].double().abs().sum(0).max())
            within(out[lo:lo + r], want, attend_bound(mean, slack, n, self.d, self.t) + small, self.t)
            got = lse[lo:lo + r].double().cpu()
            seen = torch.isfinite(want_lse)
            assert torch.equal(torch.isfinite(got), seen) and bool((got[~seen] == -math.inf).all())
            tol = (self.d + 16) * 2.0 ** -24 * slack + 2.0 ** -20 * slack + (n / 16 + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * want_lse.abs()
            assert bool(((got - want_lse).abs()[seen] <= tol[seen]).all()), float((got - want_lse).abs()[seen].max())


# How the attention kernels cut a launch into runs, one per CTA, restated from their sources: what a test's batch makes them do.

def plan_tc(rows, lens, group, kv_heads, window, sms):
    """The tensor-memory kernel's pieces: (CTA, pairs of the cell's block, tiles of the piece, tiles of the cell, cell)."""
    tile, block, cost, snap = 128, 256, 3, 1
    cells = []  # (pairs, tiles), in the launch's order
    for r, n in zip(rows, lens):
        of_head = []
        for p0 in range(0, r * group, block):
            p1 = min(r * group, p0 + block)
            first, last = n - r + p0 // group, n - r + (p1 - 1) // group
            hi = max(0, last + 1)
            lo = first + 1 - window if window and first >= window else 0
            of_head.append((p1 - p0, max(1, -(-hi // tile) - lo // tile) if hi > lo else 1))
        cells += of_head * kv_heads
    starts = np.cumsum([0] + [t + cost for _, t in cells]).tolist()
    total = starts[-1]
    per = max(1, -(-total // sms))
    snap = min(snap, per // 2)

    def cut(pos):
        if pos >= total:
            return total
        c = int(np.searchsorted(starts, pos, side="right")) - 1
        left = pos - starts[c]
        return starts[c] if left <= snap else starts[c + 1] if left + snap >= cells[c][1] else pos

    pieces = []
    for cta in range(sms):
        lo, hi = cut(cta * per), cut((cta + 1) * per)
        for c in range(len(cells)):
            a, b = max(lo, starts[c]), min(hi, starts[c] + cells[c][1])
            if a < b:
                pieces.append((cta, cells[c][0], b - a, cells[c][1], c))
    return pieces


def plan_stream(rows, lens, group, kv_heads, window, block, ctas):
    """The streaming kernel's pieces: (CTA, tiles of the piece, tiles of the cell); ``block``: pairs of a cell."""
    tile, cost, least = 64, 3, 2
    cells = []
    for r, n in zip(rows, lens):
        pos0 = n - r
        lo = (pos0 + 1 - window) // tile if window and pos0 >= window else 0
        cells += [max(1, -(-n // tile) - lo)] * (-(-r * group // block) * kv_heads)
    starts = np.cumsum([0] + [t + cost for t in cells]).tolist()
    per = max(least, -(-starts[-1] // ctas))
    pieces = []
    for cta in range(ctas):
        for c in range(len(cells)):
            a, b = max(cta * per, starts[c]), min((cta + 1) * per, starts[c] + cells[c])
            if a < b:
                pieces.append((cta, b - a, cells[c]))
    return pieces
