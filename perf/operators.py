"""Timed cases of the attention operators that read the whole K/V cache, and of the eviction that shortens it.

Three operators, each through the public calls of ``pqhsa_release_amd.ops``:

* ``decode``: one new token per sequence attends over its whole cache (``ops.DenseAttendCall``),
* ``prompt``: the rows of packed prompts, or of prompts that continue a cached one (``ops.prompt_attend``),
* ``evict``: the keys with the most accumulated attention weight are kept and copied to new pages
  (``ops.evict``).

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DIM = 128
SCALE = 1.0 / math.sqrt(DIM)
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST_PROMPT = 16384          # rows of the largest prompt: bounds what a drawn prompt may cost
LARGEST_CACHE = 4 * 8 * 131072  # (sequence, KV head, key) triples of the largest cache in 2-byte types


# --------------------------------------------------------------------------- cases
def _decode(name, B, H, G, lens, dtype, *, block=16, layout="5d", softcap=0.0, window=0, prefix=0, slopes=False,
            docs=0, mass=False, decay=1.0):
    return {"name": name, "op": "decode", "B": B, "H": H, "G": G, "n_lo": lens[0], "n_hi": lens[1], "dtype": dtype,
            "block": block, "layout": layout, "softcap": softcap, "window": window, "prefix": prefix,
            "slopes": slopes, "docs": docs, "mass": mass, "decay": decay}


def _prompt(name, B, H, G, rows, past, dtype, *, block=16, layout="5d", softcap=0.0, window=0, prefix=0,
            slopes=False, docs=0, mass_rows=0, pad=0):
    return {"name": name, "op": "prompt", "B": B, "H": H, "G": G, "rows_lo": rows[0], "rows_hi": rows[1],
            "past_lo": past[0], "past_hi": past[1], "dtype": dtype, "block": block, "layout": layout,
            "softcap": softcap, "window": window, "prefix": prefix, "slopes": slopes, "docs": docs,
            "mass_rows": mass_rows, "pad": pad}


def _evict(name, B, H, lens, dtype, keep, *, sink=4, recent=64, block=16, layout="5d"):
    return {"name": name, "op": "evict", "B": B, "H": H, "n_lo": lens[0], "n_hi": lens[1], "dtype": dtype,
            "keep": keep, "sink": sink, "recent": recent, "block": block, "layout": layout}


def listed():
    return [
        # one short fp32 context of a single head, as in a unit of an evaluation: latency
        _decode("decode-1x8192-fp32", 1, 1, 1, (8192, 8192), "fp32", block=0, layout="dense"),
        # a chat service's batch of short contexts of odd lengths, capped scores
        _decode("decode-16x700-capped", 16, 8, 4, (1, 701), "bf16", softcap=30.0),
        # one 32K context, the ordinary long-context request
        _decode("decode-1x32768", 1, 8, 4, (32768, 32768), "bf16"),
        # a ragged batch that tracks the weight of each key for a later eviction, 4-D pages, seven heads a group
        _decode("decode-16x64k-mass", 16, 4, 7, (16384, 65536), "fp16", layout="4d", mass=True, decay=0.98),
        # the largest cache: 4 x 128K, every key read
        _decode("decode-4x131072", 4, 8, 4, (131072, 131072), "bf16"),
        # a short prompt of odd length in fp32, scores biased by distance
        _prompt("prompt-1x517-fp32-bias", 1, 2, 4, (517, 517), (0, 0), "fp32", slopes=True),
        # training documents or requests packed into sequences, a prefix open to all rows
        _prompt("prompt-6x1800-documents", 6, 8, 4, (300, 1801), (0, 0), "bf16", docs=5, prefix=100, pad=37),
        # 64 new rows behind a cached 32K prompt, the last rows' weights kept for an eviction
        _prompt("prompt-continue-32k", 1, 4, 7, (64, 64), (32704, 32704), "fp16", mass_rows=32),
        # a whole 16K prompt: the compute-bound end
        _prompt("prompt-1x16384", 1, 8, 4, (LARGEST_PROMPT, LARGEST_PROMPT), (0, 0), "bf16"),
        # a small cache halved after its prompt
        _evict("evict-1x8192", 1, 8, (8192, 8192), "bf16", 4096),
        # ragged contexts brought down to one budget
        _evict("evict-16x64k", 16, 8, (16384, 65536), "bf16", 8192),
        # the largest cache, a quarter kept
        _evict("evict-4x131072", 4, 8, (131072, 131072), "fp16", 32768, sink=16, recent=1024, layout="4d"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("decode", "prompt", "evict"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    H, G = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    layout = rng.choice(("5d", "5d", "4d", "dense"))
    block = 0 if layout == "dense" else rng.choice((16, 16, 24, 64, 128))
    rule = {"softcap": rng.choice((0.0, 0.0, 20.0, 50.0)), "window": rng.choice((0, 0, _log_int(rng, 1, 8192))),
            "prefix": rng.choice((0, 0, _log_int(rng, 1, 400))), "slopes": rng.random() < 0.3,
            "docs": rng.choice((0, 0, 0, rng.randint(2, 9)))}
    weight = 2 if dtype == "fp32" else 1
    if kind == "prompt":
        B = _log_int(rng, 1, 8)
        rows = _log_int(rng, 1, 8192)
        past = rng.choice((0, 0, _log_int(rng, 1, 32768)))
        # at most the largest listed prompt's products, fp32 ones counted eight times
        while B * H * G * rows * (rows + 2 * past) * (8 if dtype == "fp32" else 1) > 32 * LARGEST_PROMPT ** 2:
            rows, past, B = max(1, rows // 2), past // 2, max(1, B - 1)
        c = _prompt("", B, H, G, (max(1, rows // rng.choice((1, 2, 8))), rows), (past // 2, past), dtype, block=block,
                    layout=layout, mass_rows=rng.choice((0, 0, 1, 16, 64)), pad=rng.choice((0, 3, 50)), **rule)
    else:
        B = _log_int(rng, 1, 16)
        n = min(_log_int(rng, 1, 131072), LARGEST_CACHE // (B * H * weight))
        lens = (max(1, n // rng.choice((1, 2, 8))), n)
        if kind == "decode":
            c = _decode("", B, H, G, lens, dtype, block=block, layout=layout, mass=rng.random() < 0.4,
                        decay=rng.choice((1.0, 0.95)), **rule)
        else:
            sink, recent = rng.choice((0, 1, 4, 16)), rng.choice((0, 1, 64, 100))
            c = _evict("", B, H, lens, dtype, max(sink + recent, 1, int(n * rng.uniform(0.1, 0.6))), sink=sink,
                       recent=recent, block=block, layout=layout)
    del c["name"]
    return c


# --------------------------------------------------------------------------- inputs
def _lens(rng, lo, hi, count):
    """The longest first, so that the bound a program knows on the host is the case's own."""
    return [hi] + [rng.randint(lo, hi) for _ in range(count - 1)]


def _cache(case, gen, lens, caps):
    """K and V of a cache and where each token of a sequence lies: (tensors a program holds, table, slots).

    Keys are Gaussian with a scale of its own for every channel, values Gaussian."""
    B, H, block, dt = case["B"], case["H"], case["block"], DTYPES[case["dtype"]]
    channel = torch.exp(0.5 * torch.randn(DIM, generator=gen, device="cuda")).to(dt)
    if case["layout"] == "dense":
        k = torch.randn(B, H, max(caps), DIM, generator=gen, device="cuda", dtype=dt).mul_(channel)
        v = torch.randn(B, H, max(caps), DIM, generator=gen, device="cuda", dtype=dt)
        return {"k": k, "v": v, "table": None}
    per = [-(-c // block) for c in caps]
    order = torch.randperm(sum(per), generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(B, max(per), dtype=torch.int32, device="cuda")
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at : at + p]
        at += p
    if case["layout"] == "5d":
        cache = torch.randn(2, sum(per), block, H, DIM, generator=gen, device="cuda", dtype=dt)
        cache[0].mul_(channel)
        k, v = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    else:
        cache = torch.randn(sum(per), H, block, 2 * DIM, generator=gen, device="cuda", dtype=dt)
        cache[..., :DIM].mul_(channel)
        k, v = cache[..., :DIM], cache[..., DIM:]
    return {"cache": cache, "k": k, "v": v, "table": table}  # k, v: [pages, H, block, 128] views


def _empty_cache(case, caps):
    """A zeroed cache of the case's layout with its pages in order."""
    B, H, block, dt = case["B"], case["H"], case["block"], DTYPES[case["dtype"]]
    if case["layout"] == "dense":
        k = torch.zeros(B, H, max(caps), DIM, device="cuda", dtype=dt)
        return {"k": k, "v": torch.zeros_like(k), "table": None}
    per = -(-max(caps) // block)
    table = torch.arange(B * per, dtype=torch.int32, device="cuda").reshape(B, per)
    if case["layout"] == "5d":
        cache = torch.zeros(2, B * per, block, H, DIM, device="cuda", dtype=dt)
        k, v = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    else:
        cache = torch.zeros(B * per, H, block, 2 * DIM, device="cuda", dtype=dt)
        k, v = cache[..., :DIM], cache[..., DIM:]
    return {"cache": cache, "k": k, "v": v, "table": table}


def _rows_of(s, which, seq, head, pos):
    """Rows of a cache by index tensors that broadcast against each other."""
    t = s["kv"][which] if which in ("k", "v") else which
    if s["kv"]["table"] is None:
        return t[seq, head, pos]
    block = s["block"]
    return t[s["kv"]["table"][seq, pos // block].long(), head, pos % block]


def _rule_inputs(case, rng, gen, lens):
    B, n_max = case["B"], max(lens)
    r = {"slopes": None, "prefix": None, "docs": None}
    if case["slopes"]:  # a geometric series over the query heads, as models with distance biases use
        heads = case["H"] * case["G"]
        r["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device="cuda")
    if case["prefix"]:
        r["prefix"] = torch.tensor([rng.randint(0, case["prefix"]) for _ in range(B)], dtype=torch.int32, device="cuda")
    if case["docs"]:
        docs = torch.zeros(B, n_max, dtype=torch.int32)
        for b, n in enumerate(lens):
            cuts = sorted(rng.randint(1, n) for _ in range(case["docs"] - 1))
            ids = torch.zeros(n + 1, dtype=torch.int32)
            for c in cuts:
                ids[c] += 1
            docs[b, :n] = ids[:n].cumsum(0).to(torch.int32)
        r["docs"] = docs.cuda()
    return r


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, dt = case["B"], case["H"], DTYPES[case["dtype"]]
    s = {"case": case, "op": case["op"], "block": case["block"]}
    if case["op"] == "evict":
        return _prepare_evict(case, rng, gen, s)
    G = case["G"]
    if case["op"] == "decode":
        rows = [1] * B
        lens = _lens(rng, case["n_lo"], case["n_hi"], B)
    else:
        # the same rows for every seed, so that the packed batch has one size
        rows = _lens(random.Random(B), case["rows_lo"], case["rows_hi"], B)
        lens = [r + p for r, p in zip(rows, _lens(rng, case["past_lo"], case["past_hi"], B))]
    s["lens"], s["rows"], s["n_max"] = lens, rows, max(lens)
    s["kv"] = _cache(case, gen, lens, lens)
    s["rule"] = _rule_inputs(case, rng, gen, lens)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    s["cu_rows"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    total = cu[-1] + case.get("pad", 0)
    # a query row is one of the keys it sees, a little shortened, with noise: a few keys stand out
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(rows, device="cuda"))
    at = torch.arange(cu[-1], device="cuda") - s["cu_rows"][seq].long() + s["seq_lens"][seq].long() - torch.tensor(rows, device="cuda")[seq]
    pick = (torch.rand(cu[-1], H, G, generator=gen, device="cuda") * (at + 1).reshape(-1, 1, 1)).long()
    pick = torch.minimum(pick, at.reshape(-1, 1, 1))
    q = 0.2 * torch.randn(total, H, G, DIM, generator=gen, device="cuda")
    q[: cu[-1]] += 0.7 * _rows_of(s, "k", seq.reshape(-1, 1, 1), torch.arange(H, device="cuda").reshape(1, H, 1), pick).float()
    s["q"] = q.reshape(total, H * G, DIM).to(dt)
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(total, H * G, device="cuda")
    s["mass"] = s["mass_in"] = None
    if case.get("mass"):
        s["mass_in"] = torch.rand(B, H, s["n_max"], generator=gen, device="cuda")
        s["mass"] = torch.zeros_like(s["mass_in"])
    elif case.get("mass_rows"):
        s["mass"] = torch.zeros(B, H, s["n_max"], device="cuda")
    if own:
        from pqhsa_release_amd import ops

        kv = s["kv"]
        s["source"] = ops.kv_contiguous(kv["k"], kv["v"]) if kv["table"] is None else ops.kv_paged(kv["cache"], kv["table"])
        s["score"] = ops.ScoreRule(scale=SCALE, softcap=case["softcap"], window=case["window"], **s["rule"])
        if case["op"] == "decode":
            s["call"] = ops.DenseAttendCall(s["q"], s["out"], s["source"], G, s["seq_lens"], n_max=s["n_max"], rule=s["score"],
                                            lse=s["lse"], mass=s["mass"], mass_in=s["mass_in"], decay=case["decay"])
    return s


def _prepare_evict(case, rng, gen, s):
    B, H, keep = case["B"], case["H"], case["keep"]
    lens = _lens(rng, case["n_lo"], case["n_hi"], B)
    s["lens"], s["n_max"] = lens, max(lens)
    s["kv"] = _cache(case, gen, lens, lens)
    s["dst"] = _empty_cache(case, [keep] * B)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # accumulated weights have a heavy tail, and many keys that no row looked at hold exactly nothing
    mass = torch.exp(3.0 * torch.randn(B, H, s["n_max"], generator=gen, device="cuda") - 6.0)
    s["mass"] = mass * (torch.rand(B, H, s["n_max"], generator=gen, device="cuda") > 0.3)
    s["mass_out"] = torch.zeros(B, H, keep, device="cuda")
    if own:
        from pqhsa_release_amd import ops

        for name in ("kv", "dst"):
            kv = s[name]
            s[name + "_source"] = ops.kv_contiguous(kv["k"], kv["v"]) if kv["table"] is None else ops.kv_paged(kv["cache"], kv["table"])
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if s["op"] == "evict":
        return _run_evict(s)
    if own:
        from pqhsa_release_amd import ops

        if s["op"] == "decode":
            s["call"].run()
        else:
            ops.prompt_attend(s["q"], s["out"], s["source"], c["G"], s["cu_rows"], s["seq_lens"], rows_max=max(s["rows"]),
                              n_max=s["n_max"], rule=s["score"], lse=s["lse"], mass=s["mass"], mass_rows=c["mass_rows"])
        got = {"out": s["out"], "lse": s["lse"]}
        if s["mass"] is not None:
            got["mass"] = s["mass"]
        return got
    return _plain_attend(s)


def _plain_attend(s):
    c = s["case"]
    B, H, G, n, dev = c["B"], c["H"], c["G"], s["n_max"], s["q"].device
    heads = torch.arange(H, device=dev)
    key_pos = torch.arange(n, device=dev)
    seq = torch.arange(B, device=dev)
    held = key_pos.reshape(1, n) < s["seq_lens"].reshape(B, 1)
    at = torch.where(held, key_pos, 0)
    K = _rows_of(s, "k", seq.reshape(B, 1, 1), heads.reshape(1, H, 1), at.reshape(B, 1, n)).float()
    V = _rows_of(s, "v", seq.reshape(B, 1, 1), heads.reshape(1, H, 1), at.reshape(B, 1, n)).float()
    # rows of every sequence side by side, the shorter ones filled up with rows that see nothing
    R = max(s["rows"])
    count = (s["cu_rows"][1:] - s["cu_rows"][:-1]).long().reshape(B, 1)
    r = torch.arange(R, device=dev).reshape(1, R)
    live = r < count
    row = torch.where(live, s["cu_rows"][:-1].long().reshape(B, 1) + r, 0)
    pos = s["seq_lens"].long().reshape(B, 1) - count + r
    q = s["q"].float()[row].reshape(B, R, H, G, DIM).permute(0, 2, 3, 1, 4).reshape(B, H, G * R, DIM)
    z = torch.matmul(q, K.transpose(2, 3).contiguous()).mul_(SCALE).reshape(B, H, G, R, n)
    if c["softcap"]:
        z.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    i, j = pos.reshape(B, R, 1), key_pos.reshape(1, 1, n)
    if c["slopes"]:
        z -= s["rule"]["slopes"].reshape(1, H, G, 1, 1) * (i - j).abs().float().reshape(B, 1, 1, R, n)
    see = j <= i
    if c["window"]:
        see = see & (i - j < c["window"])
    if s["rule"]["prefix"] is not None:
        see = see | (j < s["rule"]["prefix"].reshape(B, 1, 1))
    if s["rule"]["docs"] is not None:
        ids = s["rule"]["docs"]
        see = see & (torch.gather(ids, 1, pos.clamp(0, n - 1)).reshape(B, R, 1) == ids.reshape(B, 1, n))
    see = see & live.reshape(B, R, 1) & held.reshape(B, 1, n) & (i >= 0)
    z.masked_fill_(~see.reshape(B, 1, 1, R, n), -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    z.sub_(top).exp_()
    total = z.sum(-1, keepdim=True)
    z.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(z.reshape(B, H, G * R, n), V).reshape(B, H, G, R, DIM).permute(0, 3, 1, 2, 4).reshape(B, R, H * G, DIM)
    lse = (top + torch.log(total)).reshape(B, H, G, R).permute(0, 3, 1, 2).reshape(B, R, H * G)
    out, out_lse = torch.zeros_like(s["q"]), torch.zeros_like(s["lse"])
    out[row[live]] = o[live].to(out.dtype)
    out_lse[row[live]] = lse[live]
    got = {"out": out, "lse": out_lse}
    if s["mass"] is not None:
        if c.get("mass_rows"):
            z *= (r >= count - c["mass_rows"]).reshape(B, 1, 1, R, 1)
        mass = z.sum((2, 3))
        if s["mass_in"] is not None:
            mass += c["decay"] * s["mass_in"]
        got["mass"] = torch.where(held.reshape(B, 1, n), mass, 0.0)
    return got


def _run_evict(s):
    c = s["case"]
    if own:
        from pqhsa_release_amd import ops

        kept, lens = ops.evict(s["kv_source"], s["dst_source"], s["mass"], s["seq_lens"], keep=c["keep"], sink=c["sink"],
                               recent=c["recent"], n_max=s["n_max"], mass_out=s["mass_out"])
        dst = s["dst"]
        return {"kept": kept, "lens": lens, "mass": s["mass_out"], "k": dst["k"], "v": dst["v"]}
    B, H, n, keep, dev = c["B"], c["H"], s["n_max"], c["keep"], s["mass"].device
    lens = s["seq_lens"].long().reshape(B, 1, 1)
    pos = torch.arange(n, device=dev).reshape(1, 1, n)
    # the first and the last keys stay, the others by their weight, equal ones from the front
    must = (pos < c["sink"]) | (pos >= lens - c["recent"])
    weight = torch.where(must, math.inf, s["mass"])
    weight = torch.where(pos < lens, weight, -math.inf)
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices[..., :keep]
    new = s["seq_lens"].clamp(max=keep).long().reshape(B, 1, 1)
    slot = torch.arange(order.shape[-1], device=dev).reshape(1, 1, -1)
    kept = torch.sort(torch.where(slot < new, order, n), dim=-1).values
    live = slot < new
    at = torch.where(live, kept, 0)
    mass = torch.where(live, torch.gather(s["mass"], 2, at), 0.0)
    full = torch.full((B, H, keep), -1, dtype=torch.int32, device=dev)
    full[..., : at.shape[-1]] = torch.where(live, kept, -1).to(torch.int32)
    mass_out = torch.zeros_like(s["mass_out"])
    mass_out[..., : at.shape[-1]] = mass
    seq, head = torch.arange(B, device=dev).reshape(B, 1, 1), torch.arange(H, device=dev).reshape(1, H, 1)
    got = {"kept": full, "lens": new.reshape(B).to(torch.int32), "mass": mass_out}
    where = torch.nonzero(live.expand(B, H, -1), as_tuple=True)
    for name in ("k", "v"):
        rows = _rows_of(s, name, seq, head, at)[where]
        dst, table = torch.zeros_like(s["dst"][name]), s["dst"]["table"]
        if table is None:
            dst[where] = rows
        else:
            dst[table[where[0], where[2] // c["block"]].long(), where[1], where[2] % c["block"]] = rows
        got[name] = dst
    return got


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    B, H, size = c["B"], c["H"], 4 if c["dtype"] == "fp32" else 2
    row = 2 * DIM * size  # a key and its value

    def mean(lo, hi):  # per sequence: the longest, and the others evenly spread
        return (hi + (B - 1) * (lo + hi) / 2) / B

    if c["op"] == "evict":
        n = mean(c["n_lo"], c["n_hi"])
        kept = min(c["keep"], n)
        return {"bytes": B * H * (4 * n + kept * (2 * row + 12)), "flops": B * H * n}
    heads = H * c["G"]
    rows = 1 if c["op"] == "decode" else mean(c["rows_lo"], c["rows_hi"])
    n = mean(c["n_lo"], c["n_hi"]) if c["op"] == "decode" else rows + mean(c["past_lo"], c["past_hi"])
    first = n - rows

    def seen(upto):  # keys that a row at this position sees
        span = upto / ((c["docs"] + 1) / 2) if c["docs"] else upto
        return min(span, c["window"] + c["prefix"] / 2) if c["window"] else span

    pairs = B * rows * (seen(first + 1) + seen(n)) / 2
    read = min(n, seen(n) + rows) if c["window"] else n
    if c["op"] == "decode":
        read = seen(n)
    nbytes = B * (H * read * row + rows * heads * (2 * DIM * size + 4))
    if c.get("mass"):
        nbytes += B * H * n * 8
    flops = 4.0 * DIM * heads * pairs
    if c.get("mass_rows"):
        nbytes += B * H * n * 4
        flops += 2.0 * DIM * heads * B * min(rows, c["mass_rows"]) * n
    return {"bytes": float(nbytes), "flops": float(flops)}


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_evict(case, s) if case["op"] == "evict" else _exact_attend(case, s)


def _exact_attend(c, s):
    """One sequence, one KV head and some of its rows at a time."""
    H, G = c["H"], c["G"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    mass = None if s["mass"] is None else torch.zeros(s["mass"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (rows, n) in enumerate(zip(s["rows"], s["lens"])):
        j = torch.arange(n, device="cuda")
        step = max(1, (1 << 27) // (n * G))
        for h in range(H):
            where = torch.full_like(j, b), torch.full_like(j, h), j
            K, V = _rows_of(s, "k", *where).double(), _rows_of(s, "v", *where).double()
            for lo in range(0, rows, step):
                hi = min(rows, lo + step)
                i = torch.arange(n - rows + lo, n - rows + hi, device="cuda")
                dist = i[:, None] - j[None, :]
                ok = dist >= 0
                if c["window"]:
                    ok = torch.logical_and(ok, dist < c["window"])
                if s["rule"]["prefix"] is not None:
                    ok = torch.logical_or(ok, (j < int(s["rule"]["prefix"][b]))[None, :])
                if s["rule"]["docs"] is not None:
                    ids = s["rule"]["docs"][b]
                    ok = torch.logical_and(ok, ids[i][:, None] == ids[:n][None, :])
                for g in range(G):
                    x = s["q"][first + lo : first + hi, h * G + g].double() @ K.T / math.sqrt(DIM)
                    if c["softcap"]:
                        x = torch.tanh(x / c["softcap"]) * c["softcap"]
                    if c["slopes"]:
                        x = x - float(s["rule"]["slopes"][h * G + g]) * dist.abs()
                    x = torch.where(ok, x, torch.full_like(x, -math.inf))
                    log_total = torch.logsumexp(x, dim=1)
                    w = torch.exp(x - log_total[:, None])
                    out[first + lo : first + hi, h * G + g] = w @ V
                    lse[first + lo : first + hi, h * G + g] = log_total
                    if mass is not None:
                        last = c.get("mass_rows", 0) or rows
                        mass[b, h, :n] += w[i >= n - last].sum(0)
            if mass is not None and s["mass_in"] is not None:
                mass[b, h, :n] += c["decay"] * s["mass_in"][b, h, :n].double()
        first += rows
    return {"out": out, "lse": lse} if mass is None else {"out": out, "lse": lse, "mass": mass}


def _exact_evict(c, s):
    """The kept set from one sort by (weight, position) of every head's evictable keys."""
    import numpy as np

    B, H, keep = c["B"], c["H"], c["keep"]
    kept = np.full((B, H, keep), -1, dtype=np.int64)
    mass_out = np.zeros((B, H, keep))
    mass = s["mass"].double().cpu().numpy()
    k, v = s["dst"]["k"].double(), s["dst"]["v"].double()
    lens = []
    for b, n in enumerate(s["lens"]):
        lens.append(min(n, keep))
        low, high = min(c["sink"], n), max(min(c["sink"], n), n - c["recent"])
        for h in range(H):
            at = np.arange(n)
            if n > keep:
                middle = np.arange(low, high)
                order = np.lexsort((middle, -mass[b, h, low:high]))
                best = np.sort(middle[order[: keep - low - (n - high)]])
                at = np.concatenate([np.arange(low), best, np.arange(high, n)])
            kept[b, h, : len(at)] = at
            mass_out[b, h, : len(at)] = mass[b, h, at]
            pos = torch.from_numpy(at).cuda()
            slot = torch.arange(len(at), device="cuda")
            for name, dst in (("k", k), ("v", v)):
                rows = _rows_of(s, name, torch.full_like(pos, b), torch.full_like(pos, h), pos).double()
                if s["dst"]["table"] is None:
                    dst[b, h, : len(at)] = rows
                else:
                    dst[s["dst"]["table"][b, slot // c["block"]].long(), h, slot % c["block"]] = rows
    return {"kept": kept, "lens": np.array(lens), "mass": mass_out, "k": k, "v": v}
