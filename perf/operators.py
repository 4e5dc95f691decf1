"""The paged-cache operators: what they compute in plain torch operations, and the cases they are measured on.

Three operators, used one after the other in a layer of a served model:

  rope    head rows of Q or K rotated at their positions, adjacent or half-split pairs, part of the head, with a
          frequency table that may be scaled for long contexts; or the gradient of that (the inverse rotation)
  append  a batch of sequences' new K and V rows stored into the pages of their cache, K rotated on the way, and the
          same call's Q rows rotated too
  attend  the batch's query rows (one per sequence, a block to verify, or a chunk of a prompt) over the pages

A batch is ragged: sequence s owns the rows [row_start[s], row_start[s + 1]) of the packed row tensors, its cache
holds kv_len[s] keys once its new rows are stored, so its row i sits at position kv_len[s] - rows + i, and the key of
position p lies in page table[s][p // page_size], row p % page_size.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: the type the pages hold for each type of the rows: f32 rows are rounded to half on their way in
_PAGE_TYPES = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ------------------------------------------------------------------------------------------------------

def _rope(name, dtype, rows, heads, d, rotary, pairing, scaling, far, inverse):
    return {"name": name, "op": "rope", "dtype": dtype, "rows": rows, "heads": heads, "head_dim": d, "rotary": rotary,
            "pairing": pairing, "scaling": scaling, "far": far, "inverse": inverse}


def _append(name, dtype, seqs, rows_lo, rows_hi, len_lo, len_hi, hq, hkv, d, rotary, pairing, page, layout):
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "rows_lo": rows_lo, "rows_hi": rows_hi,
            "len_lo": len_lo, "len_hi": len_hi, "q_heads": hq, "kv_heads": hkv, "head_dim": d, "rotary": rotary,
            "pairing": pairing, "page": page, "layout": layout}


def _attend(name, dtype, seqs, rows_lo, rows_hi, len_lo, len_hi, hq, hkv, d, page, layout, window):
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "rows_lo": rows_lo, "rows_hi": rows_hi,
            "len_lo": len_lo, "len_hi": len_hi, "q_heads": hq, "kv_heads": hkv, "head_dim": d, "page": page,
            "layout": layout, "window": window}


def listed():
    return [
        # the Q rows of one decode step of 16 sequences: nothing but latency
        _rope("rope_decode", "bf16", 16, 32, 128, 128, 1, "none", 8192, False),
        # a prompt's Q rows at far positions of a stretched context: bandwidth
        _rope("rope_prompt", "bf16", 8192, 64, 128, 128, 1, "bands", 131072, False),
        # the gradient of a rotation of adjacent pairs over part of an odd-sized block's heads
        _rope("rope_gradient", "f32", 1537, 33, 96, 64, 0, "linear", 32768, True),
        # one token for each of 16 resident sequences (the continuous-batching configuration), f32 rows into half pages
        _append("append_decode", "f32", 16, 1, 1, 256, 8192, 32, 8, 128, 128, 1, 16, "head"),
        # ragged prompt chunks arriving together, pages ending inside them
        _append("append_prompt", "bf16", 6, 611, 2048, 611, 6000, 64, 8, 128, 128, 1, 32, "token"),
        # one long sequence's decode step: f32 rows over half pages, context 4096
        _attend("decode_single", "f32", 1, 1, 1, 4096, 4096, 32, 8, 128, 16, "head", 0),
        # 16 resident sequences of ragged lengths, one token each
        _attend("decode_ragged", "bf16", 16, 1, 1, 256, 8192, 32, 8, 128, 16, "token", 0),
        # one layer of the long-context decode configuration: 1 GiB of keys and values
        _attend("decode_long", "f32", 8, 1, 1, 32768, 32768, 64, 8, 128, 64, "head", 0),
        # 16 sessions verifying 7 drafted tokens each behind a shared-length prefix
        _attend("verify", "f16", 16, 7, 7, 2055, 2487, 32, 8, 128, 16, "head", 0),
        # small-headed model, sliding window, ragged chunks of odd lengths
        _attend("chunk_window", "bf16", 5, 129, 1000, 700, 5001, 32, 4, 64, 32, "token", 1024),
        # prompt ingestion in the framework's own row type: 4 sessions x 512 rows
        _attend("chunk_f32", "f32", 4, 512, 512, 1024, 2048, 32, 8, 128, 64, "head", 0),
        # one prompt's chunk deep inside a long context: matrix products
        _attend("chunk_long", "bf16", 1, 4096, 4096, 16384, 16384, 32, 8, 128, 64, "head", 0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["f32", "f16", "bf16"])
    d = rng.choice([64, 64, 96, 128, 128, 128, 256])
    rotary = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
    pairing = rng.randint(0, 1)
    op = rng.choice(["rope", "append", "attend", "attend"])
    if op == "rope":
        heads, rows = rng.randint(1, 64), spread(1, 8192)
        c = _rope("", dtype, rows, heads, min(d, 128), min(rotary, 128), pairing,
                  rng.choice(["none", "linear", "bands", "ramp"]), spread(512, 131072), rng.random() < 0.4)
        while c["rows"] * c["heads"] * (4 if dtype == "f32" else 2) > 8192 * 64 * 2:
            c["rows"] = (c["rows"] + 1) // 2
    else:
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
        group = rng.choice([1, 2, 4, 4, 7, 8])
        group = min(group, 64 // kv_heads)
        page = rng.choice([8, 16, 16, 32, 64, 128])
        layout = rng.choice(["head", "token"])
        seqs = spread(1, 48)
        len_hi = spread(16, 16384)
        len_lo = spread(1, len_hi)
        if op == "append":
            rows_hi = min(len_lo, spread(1, 2048))
            rows_lo = rng.randint(0, rows_hi)
            while seqs > 1 and (seqs * rows_hi * kv_heads * group > 6 * 1400 * 64 or seqs * len_hi * kv_heads * d > 1 << 27):
                seqs = seqs // 2
            c = _append("", dtype, seqs, rows_lo, rows_hi, len_lo, len_hi, kv_heads * group, kv_heads, d, rotary, pairing,
                        page, layout)
        else:
            kind = rng.choice(["decode", "verify", "chunk"])
            rows_hi = min(len_lo, 1 if kind == "decode" else rng.randint(2, 16) if kind == "verify" else spread(17, 4096))
            rows_lo = rows_hi if kind == "decode" else rng.randint(0, rows_hi)
            while seqs > 1 and (seqs * rows_hi * kv_heads * group * len_hi > 1 << 30 or seqs * len_hi * kv_heads * d > 1 << 27):
                seqs = seqs // 2
            while rows_hi * kv_heads * group * len_hi * d > 4096 * 32 * 13000 * 128:
                rows_hi = rows_hi // 2
                rows_lo = min(rows_lo, rows_hi)
            window = 0 if rng.random() < 0.7 else spread(1, 2 * len_hi)
            c = _attend("", dtype, seqs, rows_lo, rows_hi, len_lo, len_hi, kv_heads * group, kv_heads, d, page, layout, window)
    del c["name"]
    return c


def _ragged(case):
    """(rows, keys) of every sequence: spread evenly over the case's ranges, in an order of their own."""
    n = case["seqs"]

    def between(lo, hi, step):
        return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)] if n > 1 else [hi]

    # a stride without a common factor with n visits every value of the range once
    step = next((s for s in (7, 5, 3) if math.gcd(s, n) == 1), 1)
    return between(case["rows_lo"], case["rows_hi"], 1), between(case["len_lo"], case["len_hi"], step)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["head_dim"] * size + 4 * case["rows"], "flops": 3 * n * case["rotary"]}
    rows, keys = _ragged(case)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    total = sum(rows)
    if case["op"] == "append":
        return {"bytes": total * d * (size * (2 * hq + 2 * hkv) + 2 * 2 * hkv), "flops": 3 * total * (hq + hkv) * case["rotary"]}
    read = pairs = 0
    for r, n in zip(rows, keys):
        w = case["window"] or n
        read += min(n, r - 1 + w) if r else 0
        # the rows' positions are n - r .. n - 1; a row at position p sees min(p + 1, w) keys
        short = max(0, min(r, w - (n - r)))  # rows that see fewer than w keys, or just as many
        pairs += short * (n - r) + short * (short + 1) // 2 + (r - short) * w
    return {"bytes": read * hkv * d * 2 * 2 + 2 * total * hq * d * size + 4 * total * hq, "flops": 4 * d * hq * pairs}


# ---- what a user's program has in hand ----------------------------------------------------------------------------------

def _frequencies(rotary, scaling):
    """The rotation's angle per position of each pair, in 64 bits: base^(-2i / rotary), scaled for a context that is
    8 times the trained one - every frequency ("linear"), or the slow ones only with a smooth passage between two wave
    lengths ("bands") or between two pair numbers ("ramp") - and the factor on cosine and sine that goes with it."""
    i = torch.arange(rotary // 2, dtype=torch.float64)
    f = 500000.0 ** (-2.0 * i / rotary)
    if scaling == "linear":
        return f / 8.0, 1.0
    if scaling == "bands":
        turns = 8192.0 * f / (2 * math.pi)  # over the trained context
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * (keep + (1 - keep) / 8.0), 1.0
    if scaling == "ramp":
        def pair_of(turns):
            return rotary * math.log(8192.0 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))

        low, high = max(0.0, math.floor(pair_of(32.0))), min(rotary / 2 - 1.0, math.ceil(pair_of(1.0)))
        keep = 1 - ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f * (keep + (1 - keep) / 8.0), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def normal(*shape, dtype=t):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    s = dict(case)
    if case["op"] == "rope":
        s["x"] = normal(case["rows"], case["heads"], case["head_dim"])
        s["out"] = torch.empty_like(s["x"])
        # positions of a block's rows need not follow one another
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=gen, device=dev, dtype=torch.int32)
        f, s["magnitude"] = _frequencies(case["rotary"], case["scaling"])
        s["inv_freq"] = f.to(dev)
        return s
    rows, keys = _ragged(case)
    hq, hkv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    total, held = max(1, starts[-1]), [-(-n // page) for n in keys]
    n_pages, width = sum(held) + 3, max(held) + 1
    # the pages of a sequence lie anywhere in the pool; entries behind its last page hold no page's number
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    first = torch.tensor([sum(held[:i]) for i in range(len(held))], device=dev)
    count = torch.tensor(held, device=dev)
    column = torch.arange(width, device=dev)
    table = order[(first[:, None] + column).clamp(max=n_pages - 1)]
    s["table"] = torch.where(column < count[:, None], table, torch.full_like(table, -1)).contiguous()
    s["row_start"] = torch.tensor(starts, device=dev, dtype=torch.int32)
    s["kv_len"] = torch.tensor(keys, device=dev, dtype=torch.int32)
    s["max_rows"], s["max_len"] = max(rows), max(keys)
    shape = (n_pages, hkv, page, d) if case["layout"] == "head" else (n_pages, page, hkv, d)
    s["k_pool"], s["v_pool"] = (normal(*shape, dtype=_PAGE_TYPES[case["dtype"]]) for _ in range(2))
    if case["op"] == "append":
        # one projection's output: a token's Q, K and V heads side by side
        qkv = normal(total, hq + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_out"] = torch.zeros(total, hq, d, device=dev, dtype=t)
        f, s["magnitude"] = _frequencies(case["rotary"], "none")
        s["inv_freq"] = f.to(dev)
    else:
        s["q"] = normal(total, hq, d)
        s["out"] = torch.zeros(total, hq, d, device=dev, dtype=t)
        s["lse"] = torch.zeros(total, hq, device=dev, dtype=torch.float32)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from itak_torch_rebuild_b200 import paged

    if s["op"] == "rope":
        return paged.rope_apply(s["x"], s["positions"], s["inv_freq"], pairing=s["pairing"], magnitude=s["magnitude"],
                                inverse=s["inverse"], out=s["out"])
    cache = s.get("cache")
    if cache is None:  # made once, when the server lays out its pools
        cache = s["cache"] = paged.PagedKv(s["k_pool"], s["v_pool"], layout=s["layout"])
    if s["op"] == "append":
        cache.append(s["k"], s["v"], s["table"], s["row_start"], s["kv_len"], q=s["q"], q_out=s["q_out"],
                     inv_freq=s["inv_freq"], pairing=s["pairing"], magnitude=s["magnitude"])
        return s["k_pool"], s["v_pool"], s["q_out"]
    cache.attention(s["q"], s["table"], s["row_start"], s["kv_len"], max_rows=s["max_rows"], window=s["window"],
                    out=s["out"], lse=s["lse"])
    return s["out"], s["lse"]


def _turn(x, positions, inv_freq, pairing, magnitude, inverse):
    """Head rows x [rows, heads, head_dim] rotated at positions [rows], in f32 with the angles in 64 bits: at 100,000
    positions an f32 angle is off by hundredths."""
    angle = positions.double()[:, None] * inv_freq
    c, n = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    n = -n if inverse else n
    half, x = inv_freq.numel(), x.float()
    if pairing == 0:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * n, a * n + b * c), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * c - b * n, a * n + b * c), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _owners(s, total):
    """Each packed row's sequence and its position there (rows behind the last sequence: the last one's, and no position)."""
    starts, kv_len = s["row_start"].long(), s["kv_len"].long()
    row = torch.arange(total, device=starts.device)
    seq = torch.searchsorted(starts[1:], row, right=True).clamp(max=kv_len.numel() - 1)
    return seq, torch.where(row < starts[-1], kv_len[seq] - (starts[seq + 1] - row), torch.full_like(row, -1))


def _run_plain(s):
    if s["op"] == "rope":
        s["out"].copy_(_turn(s["x"], s["positions"], s["inv_freq"], s["pairing"], s["magnitude"], s["inverse"]))
        return s["out"]
    page, hkv, d = s["page"], s["kv_heads"], s["head_dim"]
    total = s["q"].shape[0]
    if s["op"] == "append":
        seq, pos = _owners(s, total)
        if int(s["row_start"].numel()) and s["max_rows"]:
            at, off = s["table"].long()[seq, pos.clamp(min=0) // page], pos.clamp(min=0) % page
            k = _turn(s["k"], pos, s["inv_freq"], s["pairing"], s["magnitude"], False)
            for pool, new in ((s["k_pool"], k), (s["v_pool"], s["v"])):
                if s["layout"] == "head":
                    pool[at, :, off] = new.to(pool.dtype)
                else:
                    pool[at, off] = new.to(pool.dtype)
            s["q_out"].copy_(_turn(s["q"], pos, s["inv_freq"], s["pairing"], s["magnitude"], False))
        return s["k_pool"], s["v_pool"], s["q_out"]

    # the pages gathered into one padded block of rows, [seqs, kv_heads, keys, head_dim]
    group, rmax = s["q_heads"] // hkv, s["max_rows"]
    if rmax == 0:
        return s["out"], s["lse"]
    width = -(-s["max_len"] // page)

    def gathered(pool):
        x = pool[s["table"][:, :width].clamp(min=0).long()]
        x = x.transpose(1, 2) if s["layout"] == "head" else x.permute(0, 3, 1, 2, 4)
        return x.reshape(x.shape[0], hkv, width * page, d).float()

    keys, values = gathered(s["k_pool"]), gathered(s["v_pool"])
    starts, kv_len = s["row_start"].long(), s["kv_len"].long()
    seqs, r = kv_len.numel(), torch.arange(rmax, device=keys.device)
    q = s["q"][(starts[:-1, None] + r).clamp(max=total - 1)].float()  # [seqs, rows, q_heads, head_dim]
    q = q.reshape(seqs, rmax, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, rmax * group, d)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), keys.transpose(-1, -2)).view(seqs, hkv, rmax, group, width * page)
    at = (kv_len - (starts[1:] - starts[:-1]))[:, None] + r  # [seqs, rows] positions
    key = torch.arange(width * page, device=keys.device)
    hidden = (key > at[..., None]) | (key >= kv_len[:, None, None])
    if s["window"]:
        hidden |= key <= at[..., None] - s["window"]
    scores.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    sums = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, hkv, rmax * group, -1), values).view(seqs, hkv, rmax, group, d)
    out = torch.where(sums > 0, out / sums, torch.zeros_like(out))
    lse = torch.where(sums > 0, top + sums.log(), torch.full_like(sums, -math.inf)).squeeze(-1)
    seq, pos = _owners(s, total)
    row = (pos - (kv_len - (starts[1:] - starts[:-1]))[seq]).clamp(min=0, max=rmax - 1)
    # every packed row belongs to a sequence here, and is written whole
    s["out"].copy_(out[seq, :, row].reshape(total, s["q_heads"], d))
    s["lse"].copy_(lse[seq, :, row].reshape(total, s["q_heads"]))
    return s["out"], s["lse"]


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------

def _exact_rotation(x, positions, inv_freq, pairing, magnitude, sign):
    """Pairs as complex numbers times magnitude * exp(i * angle)."""
    n = inv_freq.numel()
    x = x.double().clone()
    first = torch.arange(n, device=x.device) * (2 if pairing == 0 else 1)
    second = first + (1 if pairing == 0 else n)
    z = torch.complex(x[..., first], x[..., second])
    angle = positions.double()[:, None] * inv_freq
    z = z * torch.polar(torch.full_like(angle, magnitude), sign * angle)[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rotation(s["x"], s["positions"], s["inv_freq"], s["pairing"], s["magnitude"], -1 if s["inverse"] else 1)
    rows, lens = _ragged(case)
    page, hkv, hq, d = s["page"], s["kv_heads"], s["q_heads"], s["head_dim"]
    head_major = s["layout"] == "head"
    if case["op"] == "append":
        k_pool, v_pool, q_out = s["k_pool"].double(), s["v_pool"].double(), s["q_out"].double()
        row = 0
        for i, (r, n) in enumerate(zip(rows, lens)):
            if r == 0:
                continue
            pos = torch.arange(n - r, n, device=k_pool.device)
            turn = (pos, s["inv_freq"], s["pairing"], s["magnitude"], 1)
            k, v = _exact_rotation(s["k"][row:row + r], *turn), s["v"][row:row + r].double()
            q_out[row:row + r] = _exact_rotation(s["q"][row:row + r], *turn)
            for pool, new in ((k_pool, k), (v_pool, v)):
                by_row = pool.transpose(1, 2) if head_major else pool
                by_row[s["table"][i, pos // page].long(), pos % page] = new
            row += r
        return k_pool, v_pool, q_out
    out, lse = s["out"].double(), s["lse"].double()
    row = 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        if r == 0:
            continue
        ids = s["table"][i, :-(-n // page)].long()
        pos = torch.arange(n - r, n, device=out.device)[:, None]
        key = torch.arange(n, device=out.device)
        seen = (key <= pos) & (key > pos - s["window"]) if s["window"] else key <= pos
        for h in range(hkv):
            k, v = ((p[ids, h] if head_major else p[ids, :, h]).reshape(-1, d)[:n].double() for p in (s["k_pool"], s["v_pool"]))
            for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                score = s["q"][row:row + r, j].double() @ k.t() / math.sqrt(d)
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                lse[row:row + r, j] = torch.logsumexp(score, -1)
                out[row:row + r, j] = torch.softmax(score, -1) @ v
        row += r
    return out, lse
