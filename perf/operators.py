"""What the 8-bit block-scaled KV cache is measured on: writing it, attending over it, evicting from it.

``run(state)`` makes one pass through one operator, in plain torch where ``own`` is false and with the calls a user
makes of ``jacq_b200.q8_cache`` where it is true.

The cache. A page holds B tokens of every kv head in 8 bits (int8, or 4-bit-exponent floats) with one fp32 scale for K
and one for V per page and head; the tokens of a sequence's last, incomplete block stay in fp16 in the sequence's tail
rows. Token j of a sequence is row j % B of logical page j // B.

The operators.

* ``write``  appends new fp16 rows, quantising every block that becomes complete (scale = largest magnitude / 127, or
  / 448 for floats; code = the value over the scale, rounded to the nearest code), then reads the rows of the blocks it
  touched back as fp16 values, which is how a sequence is handed on.
* ``attend`` softmax attention of the last q tokens of every sequence over the cache: token i sees token j <= i if
  j < sinks or j > i - window (window 0: every j <= i). With ``mass`` the softmax weights of the pass are added up per
  kv head and page.
* ``evict``  keeps ``budget`` complete pages of every sequence: the first ``first`` and last ``recent`` ones and, of the
  rest, those with the largest mass over all heads (equal ones: the lowest index), and closes up the tables.
"""
import math
import random
import zlib

import numpy as np
import torch

own = False

_TOP = {"int8": 127.0, "e4m3": 448.0}


# ---------------------------------------------------------------------------------------------- cases

def _attend(name, fmt, nkv, qpk, d, block, batch, length, **more):
    case = {"kind": "attend", "fmt": fmt, "nkv": nkv, "qpk": qpk, "d": d, "block": block, "batch": batch, "len": length,
            "shortest": length, "new": 1, "window": 0, "sinks": 0, "mass": False, **more}
    return {"name": name, **case} if name else case


def _write(name, fmt, nkv, qpk, d, block, batch, length, new, ragged, fused):
    case = {"kind": "write", "fmt": fmt, "nkv": nkv, "qpk": qpk, "d": d, "block": block, "batch": batch, "len": length,
            "shortest": 0, "new": new, "ragged": ragged, "fused": fused}
    return {"name": name, **case} if name else case


def _evict(name, nkv, block, batch, length, shortest, budget, first, recent):
    case = {"kind": "evict", "nkv": nkv, "block": block, "batch": batch, "len": length, "shortest": shortest,
            "budget": budget, "first": first, "recent": recent}
    return {"name": name, **case} if name else case


def listed():
    return [
        # a decode step of a small batch: one token a sequence, K and V slices of the fused projection's output
        _write("write_step_b8", "int8", 8, 4, 128, 16, 8, 2000, 1, False, True),
        # prompts of 1..1024 tokens arriving together behind caches of up to 100 tokens
        _write("write_prompt_b96", "e4m3", 8, 4, 128, 16, 96, 100, 1024, True, True),
        # the smallest serving step: four short sequences of the 1.1B model's heads
        _attend("decode_b4_t512", "int8", 4, 8, 64, 16, 4, 512),
        # the 0.5B model's heads, 64 sequences of unequal length, 32-token pages of 8-bit floats
        _attend("decode_b64_t4096_ragged", "e4m3", 2, 7, 64, 32, 64, 4096, shortest=1),
        # the 7B benchmark shape: 128 sequences of 8192 tokens
        _attend("decode_b128_t8192", "int8", 8, 4, 128, 16, 128, 8192),
        # one long context on the 14B model's heads, its page masses collected for eviction
        _attend("decode_mass_b1_t32768", "int8", 8, 5, 128, 16, 1, 32768, mass=True),
        # a served batch whose page masses are collected, unequal lengths
        _attend("decode_mass_b32_t6000", "e4m3", 8, 4, 128, 16, 32, 6000, shortest=500, mass=True),
        # streaming: a window and a few first tokens, long sequences
        _attend("window_decode_b48_t16384", "int8", 8, 4, 128, 16, 48, 16384, shortest=3000, window=4096, sinks=4),
        # up to eight drafted tokens a sequence are verified at once
        _attend("window_verify_b24_t8000", "int8", 8, 4, 128, 64, 24, 8000, shortest=9, new=8, window=4001, sinks=16),
        # a chunk of two prompts behind what is cached already
        _attend("window_prompt_b2_t6144", "int8", 8, 4, 128, 16, 2, 6144, shortest=5000, new=1024, window=4096, sinks=4),
        # trimming a few sequences by one page each, after a step
        _evict("evict_b4_t2048", 8, 16, 4, 2048, 2000, 120, 1, 8),
        # halving long caches of a full batch
        _evict("evict_b128_t32768", 8, 16, 128, 32768, 9000, 1024, 1, 16),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    fmt = rng.choice(("int8", "e4m3"))
    block = rng.choice((16, 16, 32, 64, 128))
    nkv, qpk = rng.choice(((1, 16), (1, 1), (2, 7), (2, 8), (4, 8), (8, 1), (8, 4), (8, 5), (5, 3), (3, 12)))
    d = rng.choice((64, 128, 128, 256))
    kind = rng.choice(("write", "attend", "attend", "attend", "evict"))
    if kind == "evict":
        batch, length = _log(rng, 1, 128), _log(rng, 200, 32768)
        full = length // block
        first, recent = rng.randrange(0, 3), rng.randrange(0, 20)
        budget = max(first + recent, 1, int(full * rng.uniform(0.2, 1.05)))
        return _evict(None, nkv, block, batch, length, rng.randrange(0, length), budget, first, recent)
    if kind == "write":
        new = _log(rng, 1, 1024)
        batch = max(1, min(_log(rng, 1, 128), 98304 * 8 * 128 // (new * nkv * d)))
        return _write(None, fmt, nkv, qpk, d, block, batch, rng.randrange(0, 3000), new, rng.random() < 0.7, rng.random() < 0.5)
    length = _log(rng, 1, 32768)
    row = 8192 * 128 * 8 * 128  # cached elements of the largest case
    batch = max(1, min(_log(rng, 1, 160), row // (2 * length * nkv * d)))
    new, window, sinks, mass = 1, 0, 0, False
    if rng.random() < 0.5:
        window, sinks = _log(rng, 1, 8192), rng.choice((0, 1, 4, 17, 128))
    if rng.random() < 0.35:
        new = min(length, _log(rng, 2, 700))
        batch = max(1, min(batch, (1 << 33) // (new * nkv * qpk * length * 16)))
    elif rng.random() < 0.4:
        mass = True
    return _attend(None, fmt, nkv, qpk, d, block, batch, length, shortest=rng.randrange(0, length + 1), new=new,
                   window=window, sinks=sinks, mass=mass)


def _lens(case):
    """Tokens a sequence holds (write: before the call) and how many are new; they go by the case alone."""
    pick = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    lens = [pick.randint(min(case["shortest"], case["len"]), case["len"]) for _ in range(case["batch"])]
    new = case.get("new", 0)
    if case["kind"] == "attend":
        fresh = [new if new == 1 else pick.randint(1, new) if new < 64 else new for _ in lens]
        if new > 1:
            fresh = [min(f, t) for f, t in zip(fresh, lens)]
    elif case["kind"] == "write":
        fresh = [pick.randint(1, new) if case["ragged"] else new for _ in lens]
    else:
        fresh = [0 for _ in lens]
    return lens, fresh


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _pairs(case, lens, fresh):
    """(query, key) pairs that are seen, and keys that any query of the sequence sees."""
    window, sinks, pairs, keys = case["window"], case["sinks"], 0, 0
    for t, n in zip(lens, fresh):
        low = max(0, t - n - window + 1) if window else 0
        keys += t - low + min(sinks, low) if t else 0
        if not window:
            pairs += n * t - n * (n - 1) // 2
            continue
        for i in range(t - n, t):
            low = max(0, i - window + 1)
            pairs += i + 1 - low + min(sinks, low)
    return max(pairs, 0), keys


def work(case):
    lens, fresh = _lens(case)
    nkv, block = case["nkv"], case["block"]
    if case["kind"] == "evict":
        pages = sum(t // block + (t % block > 0) for t in lens)
        kept = sum(min(t // block, case["budget"]) + (t % block > 0) for t in lens)
        w = _width(case, lens)
        # masses and table entries in; masses, tables and freed pages out, whole
        return {"bytes": pages * (nkv * 4 + 4) + case["batch"] * w * (nkv * 4 + 8) + 16 * case["batch"], "flops": pages * nkv + kept}
    d, qpk = case["d"], case["qpk"]
    if case["kind"] == "write":
        row = 2 * nkv * d
        codes = tail = back = old = 0
        for t, n in zip(lens, fresh):
            full = (t % block + n) // block
            codes += full * block
            tail += (t + n) % block if full else n
            old += t % block if full else 0
            back += t % block + n
        # new rows and old tail rows in, codes, scales and tail rows out; then the rows read and written as fp16
        first = sum(fresh) * row * 2 + old * row * 2 + codes * row + codes // block * nkv * 8 + tail * row * 2
        second = codes * row + (back - codes) * row * 2 + back * row * 2
        return {"bytes": first + second, "flops": 4 * row * codes}
    pairs, keys = _pairs(case, lens, fresh)
    tail = sum(min(t % block, t) for t in lens)
    nh = nkv * qpk
    moved = (keys - min(tail, keys)) * 2 * nkv * d + min(tail, keys) * 4 * nkv * d + keys // block * (nkv * 8 + 4)
    moved += sum(fresh) * nh * d * 4
    if case["mass"]:
        moved += 8 * nkv * sum(-(-t // block) for t in lens)
    return {"bytes": max(1, moved), "flops": max(1, 4 * pairs * nh * d)}


# ---------------------------------------------------------------------------------------------- inputs

def _codes(x, fmt):
    """fp16 values [..., B, D] -> codes and fp32 scales [...]."""
    x = x.float()
    scale = x.abs().amax(dim=(-2, -1)) / _TOP[fmt]
    y = x / torch.where(scale > 0, scale, 1.0)[..., None, None]
    return (y.round().clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)), scale


def _width(case, lens):
    return max(1, max(-(-(t + case.get("new", 0) * (case["kind"] == "write")) // case["block"]) for t in lens))


def _tables(case, lens, fresh, rng):
    """Every sequence's pages, scattered over the pool. The pool has one page that no table names."""
    block, width = case["block"], _width(case, lens)
    counts = [(t + (n if case["kind"] == "write" else 0)) // block for t, n in zip(lens, fresh)]
    ids = rng.permutation(sum(counts)).astype(np.int32)
    table, at = np.zeros((len(lens), width), np.int32), 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    return torch.from_numpy(table).cuda(), sum(counts)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def prepare(case, seed):
    lens, fresh = _lens(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    nkv, block, batch = case["nkv"], case["block"], case["batch"]
    tables, pages = _tables(case, lens, fresh, rng)
    width = tables.shape[1]
    s = {"case": case, "lens": lens, "tables": tables, "seq_lens": _ints(lens)}

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"] == "evict":
        # what some hundreds of steps add up to: a few heavy pages, many light ones, some never looked at
        mass = torch.exp(2.0 * randn(batch, nkv, width))
        held = torch.arange(width, device="cuda") * block < s["seq_lens"][:, None]
        seen = torch.rand(batch, width, generator=gen, device="cuda") > 0.1
        s["mass"] = mass * (held & seen)[:, None]
        return s
    d, qpk, fmt = case["d"], case["qpk"], case["fmt"]
    kind = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    for name in ("k_pages", "v_pages"):
        s[name] = torch.zeros((pages + 1, nkv, block, d), dtype=torch.uint8, device="cuda").view(kind)
    s["scales"] = torch.zeros((pages + 1, nkv, 2), dtype=torch.float32, device="cuda")
    loud = torch.ones(nkv, 1, d, device="cuda")  # a few key channels are ten times the others
    loud[:, :, torch.randperm(d, generator=gen, device="cuda")[:3]] = 10.0
    for name, way in (("k_tail", loud), ("v_tail", 1.0)):
        s[name] = (randn(batch, nkv, block, d) * way).half()
    if case["kind"] == "write":
        total = sum(fresh)
        if case["fused"]:
            qkv = randn(total, (qpk + 2) * nkv * d).half()
            s["new_k"] = qkv[:, qpk * nkv * d:(qpk + 1) * nkv * d].view(total, nkv, d)
            s["new_v"] = qkv[:, (qpk + 1) * nkv * d:].view(total, nkv, d)
        else:
            s["new_k"], s["new_v"] = randn(total, nkv, d).half(), randn(total, nkv, d).half()
        s["new_k"].mul_(loud[:, 0])
        s["fresh"], s["offsets"] = fresh, _ints(_offsets(fresh))
        first = [t - t % block for t in lens]
        rows = [t % block + n for t, n in zip(lens, fresh)]
        s["first"], s["rows"], s["row_offsets"] = _ints(first), rows, _ints(_offsets(rows))
        s["ends"] = _ints([t + n for t, n in zip(lens, fresh)])
        return s
    step = max(1, (1 << 27) // (nkv * block * d))
    for j, (name, way) in enumerate((("k_pages", loud), ("v_pages", 1.0))):
        for at in range(0, pages, step):
            n = min(step, pages - at)
            codes, scale = _codes((randn(n, nkv, block, d) * way).half(), fmt)
            s[name].view(torch.int8)[at:at + n] = codes.view(torch.int8)
            s["scales"][at:at + n, :, j] = scale
    s["q"] = randn(sum(fresh), nkv * qpk, d).half()
    s["fresh"], s["offsets"] = fresh, _ints(_offsets(fresh))
    if case["mass"]:
        held = torch.arange(width, device="cuda") * block < s["seq_lens"][:, None]
        s["mass"] = torch.rand(batch, nkv, width, generator=gen, device="cuda") * held[:, None]
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls

def _cache(s):
    """The handle a program keeps beside its tensors."""
    if "handle" not in s:
        from jacq_b200.q8_cache import Q8Cache, Q8CacheTensors, Q8Layout
        c = s["case"]
        layout = Q8Layout(c["nkv"] * c["qpk"], c["nkv"], c["d"], c["block"], c["fmt"])
        tensors = Q8CacheTensors(s["k_pages"], s["v_pages"], s["scales"], s["k_tail"], s["v_tail"])
        s["handle"] = Q8Cache.over(layout, tensors, s["tables"], s["seq_lens"])
    return s["handle"]


def _run_own(s):
    c = s["case"]
    if c["kind"] == "evict":
        from jacq_b200.q8_cache import evict_pages
        r = evict_pages(s["tables"], s["seq_lens"], s["mass"], block_size=c["block"], budget=c["budget"], first=c["first"],
                        recent=c["recent"], max_seq_len=max(s["lens"]))
        return {"tables": r.block_tables, "lens": r.seq_lens, "mass": r.page_mass, "freed": r.freed, "counts": r.freed_counts}
    cache = _cache(s)
    if c["kind"] == "write":
        cache.write(s["new_k"], s["new_v"], s["offsets"], max_new_per_seq=c["new"], max_start_seq_len=max(s["lens"]),
                    start_seq_lens=s["seq_lens"])
        k, v = cache.read(s["row_offsets"], s["first"], s["ends"], total=sum(s["rows"]), max_rows_per_seq=max(s["rows"]))
        return {"k": k, "v": v}
    out = torch.empty_like(s["q"])
    if c["new"] == 1:
        cache.attend(s["q"], out, max_seq_len=max(s["lens"]), window=c["window"], sinks=c["sinks"], page_mass=s.get("mass"))
    else:
        cache.attend(s["q"], out, max_seq_len=max(s["lens"]), window=c["window"], sinks=c["sinks"], q_offsets=s["offsets"],
                     max_q_per_seq=max(s["fresh"]))
    return {"out": out, "mass": s["mass"]} if c["mass"] else {"out": out}


# ---------------------------------------------------------------------------------------------- the plain forms

def _values(pages, scales, index):
    """fp32 values of the pages that `index` names: [*index, NKV, B, D]."""
    codes = pages.view(torch.int8)[index].view(pages.dtype)
    return codes.float() * scales[index][..., None, None]


def _plain_write(s):
    c = s["case"]
    nkv, block, d, batch = c["nkv"], c["block"], c["d"], c["batch"]
    start, total = s["seq_lens"].long(), sum(s["fresh"])
    had, n = start % block, s["offsets"].diff().long()
    blocks = -(-(block - 1 + c["new"]) // block)
    seq = torch.arange(batch, device="cuda")
    # rows from the open block's first token on: the old tail rows, then the new ones
    of = torch.repeat_interleave(seq, n, output_size=total)
    at = torch.arange(total, device="cuda") - s["offsets"].long()[of] + had[of]
    spare = s["k_pages"].shape[0] - 1
    page = torch.arange(blocks, device="cuda")
    full = (had + n) // block
    column = (start // block)[:, None] + page
    whole = page < full[:, None]
    ids = torch.where(whole, s["tables"].long().gather(1, column.clamp(max=s["tables"].shape[1] - 1)), spare)
    row = torch.arange(block, device="cuda")
    for j, (new, pages, tail) in enumerate(((s["new_k"], s["k_pages"], s["k_tail"]), (s["new_v"], s["v_pages"], s["v_tail"]))):
        rows = torch.zeros((batch, blocks * block, nkv, d), dtype=torch.float16, device="cuda")
        rows[:, :block] = torch.where((row < had[:, None])[..., None, None], tail.transpose(1, 2), 0.0)
        rows[of, at] = new
        codes, scale = _codes(rows.view(batch, blocks, block, nkv, d).transpose(2, 3), c["fmt"])
        pages.view(torch.int8)[ids] = codes.view(torch.int8)
        s["scales"][..., j][ids] = scale
        last = rows.view(batch, blocks, block, nkv, d)[seq, full.clamp(max=blocks - 1)].transpose(1, 2)
        held = (row < ((had + n) % block)[:, None])[:, None, :, None]
        tail.copy_(torch.where(held, last, tail))
    # read back
    count = sum(s["rows"])
    of = torch.repeat_interleave(seq, s["row_offsets"].diff(), output_size=count)
    pos = torch.arange(count, device="cuda") - s["row_offsets"].long()[of] + s["first"].long()[of]
    paged = pos < ((start + n) // block * block)[of]
    ids = torch.where(paged, s["tables"].long()[of, (pos // block).clamp(max=s["tables"].shape[1] - 1)], spare)
    got = []
    for j, (pages, tail) in enumerate(((s["k_pages"], s["k_tail"]), (s["v_pages"], s["v_tail"]))):
        codes = pages.view(torch.int8)[ids, :, pos % block].view(pages.dtype).float()
        value = (codes * s["scales"][..., j][ids][..., None]).half()
        got.append(torch.where(paged[:, None, None], value, tail[of, :, pos % block]))
    return {"k": got[0], "v": got[1]}


def _plain_attend(s):
    c = s["case"]
    nkv, qpk, block, d, batch = c["nkv"], c["qpk"], c["block"], c["d"], c["batch"]
    t, n = s["seq_lens"].long(), s["offsets"].diff().long()
    most, total, width = max(s["fresh"]), s["q"].shape[0], s["tables"].shape[1]
    full = t // block
    ids = s["tables"].long()
    # keys: the pages of the table, then the tail rows at the place of the open block
    spot = torch.arange(width * block, device="cuda").expand(batch, -1)
    held = spot < (full * block)[:, None]
    row = torch.arange(block, device="cuda")
    spot = torch.cat([spot, (full * block)[:, None] + row], 1)
    held = torch.cat([held, row < (t % block)[:, None]], 1)
    kv = []
    for j, (pages, tail) in enumerate(((s["k_pages"], s["k_tail"]), (s["v_pages"], s["v_tail"]))):
        x = _values(pages, s["scales"][..., j], ids).transpose(1, 2).reshape(batch, nkv, width * block, d)
        x = torch.cat([x, tail.float()], 2)
        kv.append(torch.where(held[:, None, :, None], x, 0.0))
        del x
    first = s["offsets"].long()[:-1]
    turn = torch.arange(most, device="cuda")
    here = turn < n[:, None]
    q = s["q"][(first[:, None] + turn).clamp(max=total - 1)].float().view(batch, most, nkv, qpk, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, nkv, most * qpk, d)
    at = (t - n)[:, None] + turn
    seen = held[:, None] & (spot[:, None] <= at[..., None]) & here[..., None]
    if c["window"]:
        seen &= (spot[:, None] < c["sinks"]) | (spot[:, None] > at[..., None] - c["window"])
    seen = seen[:, None, :, None]  # [batch, 1, most, 1, keys]
    score = (q @ kv[0].transpose(2, 3)).view(batch, nkv, most, qpk, -1).mul_(1.0 / math.sqrt(d))
    score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > float("-inf"), top, 0.0)).exp_()
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-30)
    out = (p.view(batch, nkv, most * qpk, -1) @ kv[1]).view(batch, nkv, most, qpk, d)
    of = torch.repeat_interleave(torch.arange(batch, device="cuda"), n, output_size=total)
    out = out.permute(0, 2, 1, 3, 4)[of, torch.arange(total, device="cuda") - first[of]].reshape(total, nkv * qpk, d).half()
    if not c["mass"]:
        return {"out": out}
    p = p.sum((2, 3))
    mass = s["mass"]
    mass += p[..., :width * block].view(batch, nkv, width, block).sum(-1)
    spot = (full.clamp(max=width - 1)[:, None, None]).expand(-1, nkv, -1)
    mass.scatter_add_(2, spot, p[..., width * block:].sum(-1, keepdim=True))
    return {"out": out, "mass": mass}


def _plain_evict(s):
    c = s["case"]
    tables, t, mass, block, width = s["tables"], s["seq_lens"].long(), s["mass"], c["block"], s["tables"].shape[1]
    full, left = (t // block)[:, None], (t % block)[:, None]
    spot = torch.arange(width, device="cuda")
    here = spot < full
    held = here & ((spot < c["first"]) | (spot >= full - c["recent"]))
    free = here & ~held
    total = mass.double().sum(1).float()
    order = total.nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).sort(dim=1, descending=True, stable=True)[1]
    order = order.gather(1, (~free).gather(1, order).to(torch.int8).sort(dim=1, stable=True)[1])
    rank = torch.empty_like(order).scatter_(1, order, spot.expand_as(order))
    keep = here & ((full <= c["budget"]) | held | (rank < c["budget"] - held.sum(1, keepdim=True)))
    kept, gone = keep.sum(1, keepdim=True), here & ~keep
    freed = gone.sum(1, keepdim=True)
    away = (~gone).to(torch.int8).sort(dim=1, stable=True)[1]
    stay = keep | ((spot == full) & (left > 0))
    order = (~stay).to(torch.int8).sort(dim=1, stable=True)[1]
    closed = mass.gather(2, order[:, None].expand_as(mass))
    return {
        "tables": torch.where(spot < kept, tables.gather(1, order), 0),
        "lens": (kept * block + left)[:, 0].int(),
        "mass": torch.where((spot < stay.sum(1, keepdim=True))[:, None], closed, 0.0),
        "freed": torch.where(spot < freed, tables.gather(1, away), -1),
        "counts": freed[:, 0].int(),
    }


def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "attend": _plain_attend, "evict": _plain_evict}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------- in 64 bits

def _round64(x, fmt):
    """The nearest code's value, x already over its scale."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    e = torch.frexp(x)[1].clamp(min=-5) - 4  # eight steps to a power of two, 2^-9 the smallest
    step = torch.ldexp(torch.ones_like(x), e)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    lens, fresh, block = s["lens"], _lens(case)[1], case["block"]
    if case["kind"] == "evict":
        t = s["mass"].double()
        out = torch.zeros_like(t)
        score = t.sum(1).cpu().tolist()
        for i, n in enumerate(lens):
            full, first, recent = n // block, case["first"], case["recent"]
            keep = list(range(full))
            if full > case["budget"]:
                fixed = [j for j in keep if j < first or j >= full - recent]
                rest = sorted((j for j in keep if first <= j < full - recent), key=lambda j: (-score[i][j], j))
                keep = sorted(fixed + rest[:case["budget"] - len(fixed)])
            keep += [full] if n % block else []
            out[i, :, :len(keep)] = t[i][:, keep]
        return {"tables": None, "lens": None, "mass": out, "freed": None, "counts": None}
    nkv, d = case["nkv"], case["d"]
    if case["kind"] == "write":
        got, at = {"k": [], "v": []}, _offsets(fresh)
        for i, t in enumerate(lens):
            for name in ("k", "v"):
                x = torch.cat([s[name + "_tail"][i, :, :t % block].transpose(0, 1), s["new_" + name][at[i]:at[i + 1]]]).double()
                full = x.shape[0] // block
                b = x[:full * block].view(full, block, nkv, d)
                scale = b.abs().amax((1, 3), keepdim=True) / _TOP[case["fmt"]]
                b = _round64(b / torch.where(scale > 0, scale, 1.0), case["fmt"]) * scale
                got[name].append(torch.cat([b.reshape(-1, nkv, d), x[full * block:]]))
        return {name: torch.cat(v) for name, v in got.items()}
    qpk, at = case["qpk"], _offsets(fresh)
    out = torch.zeros((sum(fresh), nkv * qpk, d), dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if case["mass"] else None
    for i, (t, n) in enumerate(zip(lens, fresh)):
        if not t or not n:
            continue
        full, kv = t // block, []
        for j, name in enumerate(("k", "v")):
            ids = s["tables"][i, :full].long()
            codes = s[name + "_pages"].view(torch.int8)[ids].view(s[name + "_pages"].dtype).float().double()
            x = (codes * s["scales"][ids, :, j].double()[..., None, None]).transpose(0, 1).reshape(nkv, full * block, d)
            kv.append(torch.cat([x, s[name + "_tail"][i, :, :t % block].double()], 1))
        pos = torch.arange(t, device="cuda")
        me = torch.arange(t - n, t, device="cuda")
        gap = me[:, None] - pos
        blind = gap < 0
        if case["window"]:
            blind |= (gap >= case["window"]) & (pos >= case["sinks"])
        for h in range(nkv):
            q = s["q"][at[i]:at[i + 1], h * qpk:(h + 1) * qpk].double()
            w = torch.einsum("nqd,td->nqt", q, kv[0][h]) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(blind[:, None], float("-inf")), -1)
            out[at[i]:at[i + 1], h * qpk:(h + 1) * qpk] = torch.einsum("nqt,td->nqd", w, kv[1][h])
            if mass is not None:
                w = torch.nn.functional.pad(w.sum((0, 1)), (0, -t % block))
                mass[i, h, :w.numel() // block] += w.view(-1, block).sum(1)
    return {"out": out, "mass": mass} if case["mass"] else {"out": out}
