"""Plain forms, cases and exact values of the attention cache operators.

Four operators that a decode loop runs around ``spark_b200.attention``:

* ``rotary``  - rotary positions on part of each head, interleaved or half layout, plain or scaled frequencies,
  forward and backward;
* ``append``  - new rows of the latent cache, rotated and written to their pages;
* ``pages``   - reserving, freeing, forking and compacting the pages of sequences, in all layers at once;
* ``attend``  - attention of single tokens over the paged cache: one cache row serves every head as key and value,
  with a sink logit per head, an optional sliding window and first tokens that stay visible.

``run`` computes the plain form in elementary torch operations, or, where ``own`` is true, makes the calls of
``spark_b200.rotary`` and ``spark_b200.kv_cache``.
"""

import math
import os
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash-dgx-spark_b200")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step's queries, positions near a million under stretched frequencies
        {"name": "rotary_step", "op": "rotary", "batch": 64, "seq": 1, "heads": 64, "dim": 512, "rot": 64,
         "interleaved": True, "tail": True, "scaled": True, "far": 1000000, "dtype": "bf16", "train": False},
        # a prompt's queries
        {"name": "rotary_prompt", "op": "rotary", "batch": 1, "seq": 4099, "heads": 64, "dim": 512, "rot": 64,
         "interleaved": True, "tail": True, "scaled": True, "far": 65536, "dtype": "bf16", "train": False},
        # a training step's heads of the half layout, rotated in full: the result and the gradient of the input
        {"name": "rotary_train", "op": "rotary", "batch": 2, "seq": 2047, "heads": 32, "dim": 128, "rot": 128,
         "interleaved": False, "tail": False, "scaled": False, "far": 4096, "dtype": "fp32", "train": True},
        # one new token of each of 64 sequences into its page
        {"name": "append_step", "op": "append", "rows": 64, "seqs": 64, "far": 8192, "dim": 512, "rot": 64,
         "interleaved": True, "page": 64, "dtype": "bf16"},
        # the rows of a few long prompts
        {"name": "append_prompt", "op": "append", "rows": 32771, "seqs": 5, "far": 65536, "dim": 512, "rot": 64,
         "interleaved": True, "page": 64, "dtype": "bf16"},
        # a scheduler's step: the pages of 255 sequences freed and reserved anew
        {"name": "pages_reserve", "op": "pages", "kind": "reserve", "seqs": 255, "count": 255, "pool": 32768,
         "most": 128, "layers": 1, "page": 64, "dim": 128, "dtype": "bf16"},
        # parallel samples: the children of four prompts are dropped and forked again, in all 43 layers
        {"name": "pages_fork", "op": "pages", "kind": "fork", "seqs": 96, "count": 60, "pool": 1024,
         "most": 64, "layers": 43, "page": 64, "dim": 512, "dtype": "bf16"},
        # a half-empty pool moved together, in all 43 layers
        {"name": "pages_compact", "op": "pages", "kind": "compact", "seqs": 96, "count": 48, "pool": 1024,
         "most": 64, "layers": 43, "page": 64, "dim": 512, "dtype": "bf16"},
        # one sequence: latency
        {"name": "attend_one", "op": "attend", "rows": 1, "far": 8193, "even": True, "heads": 64, "dim": 512, "page": 64,
         "window": 0, "first": 0, "sink": True, "dtype": "bf16"},
        # an ordinary ragged batch
        {"name": "attend_batch", "op": "attend", "rows": 64, "far": 8192, "even": False, "heads": 64, "dim": 512,
         "page": 64, "window": 0, "first": 0, "sink": True, "dtype": "bf16"},
        # a sliding window with four first tokens over long sequences, a quarter of the heads
        {"name": "attend_window", "op": "attend", "rows": 256, "far": 20000, "even": False, "heads": 16, "dim": 512,
         "page": 32, "window": 128, "first": 4, "sink": True, "dtype": "fp16"},
        # long contexts
        {"name": "attend_long", "op": "attend", "rows": 16, "far": 131072, "even": False, "heads": 64, "dim": 512,
         "page": 128, "window": 0, "first": 0, "sink": True, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "pages", "attend"])
    if op == "rotary":
        train = rng.random() < 0.4
        dim = rng.choice([64, 128, 192, 256, 512])
        rot = rng.choice([r for r in (32, 64, 128, dim) if r <= dim])
        heads = rng.choice([1, 3, 8, 32, 64])
        batch = rng.choice([1, 2, 5])
        seq = _log(rng, 1, 60000000 // (batch * heads * dim * (4 if train else 1)))
        return {"op": op, "batch": batch, "seq": min(seq, 20000), "heads": heads, "dim": dim, "rot": rot,
                "interleaved": rng.random() < 0.5, "tail": rng.random() < 0.5, "scaled": rng.random() < 0.5,
                "far": _log(rng, 20001, 1000000), "dtype": rng.choice(["bf16", "fp16", "fp32"]), "train": train}
    if op == "append":
        dim = rng.choice([128, 256, 512])
        return {"op": op, "rows": _log(rng, 1, 20000), "seqs": rng.randint(1, 64), "far": rng.randint(20000, 30000),
                "dim": dim, "rot": rng.choice([32, 64, 128]), "interleaved": rng.random() < 0.7,
                "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "pages":
        kind = rng.choice(["reserve", "fork", "compact"])
        if kind == "reserve":
            seqs = rng.randint(2, 256)
            return {"op": op, "kind": kind, "seqs": seqs, "count": rng.randint(1, seqs), "pool": 32768,
                    "most": rng.randint(1, 128), "layers": 1, "page": rng.choice([16, 32, 64]), "dim": 128,
                    "dtype": "bf16"}
        seqs = rng.randint(8, 96)
        return {"op": op, "kind": kind, "seqs": seqs, "count": rng.randint(2, seqs // 2 + 1),
                "pool": rng.randint(500, 1000), "most": rng.randint(4, 64), "layers": rng.randint(1, 43),
                "page": rng.choice([16, 32, 64]), "dim": rng.choice([128, 256, 512]),
                "dtype": rng.choice(["bf16", "fp16"])}
    rows = _log(rng, 1, 256)
    window = rng.choice([0, 0, rng.randint(1, 1000)])
    heads = rng.choice([1, 5, 8, 16, 32, 64, 64, 96, 128] if rows <= 64 else [8, 16, 32, 64])
    pairs = 500000 if heads > 64 else 1100000
    return {"op": op, "rows": rows, "far": _log(rng, 1, min(130000, pairs // rows)), "even": rng.random() < 0.3,
            "heads": heads,
            "dim": rng.choice([128, 256, 512, 512]), "page": rng.choice([16, 32, 64, 128]), "window": window,
            "first": rng.choice([0, rng.randint(1, 200)]) if window else 0, "sink": rng.random() < 0.7,
            "dtype": rng.choice(["bf16", "fp16"])}


# ------------------------------------------------------------------------------------------------- prepare
def _frequencies(rot, scaled):
    """Radians per position of each pair: base^(-2i/rot), or stretched 16-fold below a ramp over the pairs that turn
    between once and 32 times in 65536 positions."""
    base = 10000.0
    pair = torch.arange(rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * pair / rot)
    if scaled:
        turns = lambda n: rot * math.log(65536 / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rot - 1)
        ramp = ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / 16.0 * ramp + f * (1 - ramp)
    return f.cuda()


def _lengths(g, rows, far, even):
    """Ragged sequence lengths from 1 to `far`, spread over their logarithm, the first the longest."""
    if even:
        return torch.full((rows,), far, dtype=torch.int64, device="cuda")
    lens = torch.exp(torch.rand(rows, generator=g, device="cuda") * math.log(max(far, 2))).long().clamp(1, far)
    lens = torch.maximum(lens, torch.rand(rows, generator=g, device="cuda").mul(far).long().clamp(1, far))
    lens[0] = far
    return lens


def _table(g, lens, page, pool):
    """A page table [rows, most] over the shuffled pages of a pool."""
    need = (lens + page - 1) // page
    order = torch.randperm(pool, generator=g, device="cuda")
    slot = torch.arange(int(need.max()), device="cuda")[None]
    start = (need.cumsum(0) - need)[:, None]
    return torch.where(slot < need[:, None], order[(start + slot).clamp(max=pool - 1)], -1).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    s = {"case": case}
    if case["op"] == "rotary":
        shape = (case["batch"], case["seq"], case["heads"], case["dim"])
        s["x"] = rand(*shape).to(dt)
        start = torch.randint(0, case["far"] - case["seq"] + 1, (case["batch"], 1), generator=g, device="cuda")
        s["positions"] = start + torch.arange(case["seq"], device="cuda")[None]
        s["freqs"] = _frequencies(case["rot"], case["scaled"])
        s["offset"] = case["dim"] - case["rot"] if case["tail"] else 0
        if case["train"]:
            s["x"].requires_grad_(True)
            s["grad"] = rand(*shape).to(dt)
    elif case["op"] == "append":
        rows, seqs = case["rows"], min(case["seqs"], case["rows"])
        each = torch.full((seqs,), rows // seqs, dtype=torch.int64, device="cuda")
        each[: rows % seqs] += 1
        start = (torch.rand(seqs, generator=g, device="cuda") * (case["far"] - int(each.max()) + 1)).long()
        seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), each)
        within = torch.arange(rows, device="cuda") - (each.cumsum(0) - each)[seq]
        pool = seqs * (-(-case["far"] // case["page"])) + 7
        s["table"] = _table(g, start + each, case["page"], pool)
        s["pages"] = torch.empty(pool, case["page"], case["dim"], dtype=dt, device="cuda").normal_(generator=g)
        s["rows"] = rand(rows, case["dim"]).to(dt)
        s["seq_ids"], s["positions"] = seq.int(), (start[seq] + within).int()
        s["freqs"] = _frequencies(case["rot"], True)
    elif case["op"] == "pages":
        seqs, page, kind = case["seqs"], case["page"], case["kind"]
        far = case["most"] * page
        if kind == "reserve":
            held = (torch.rand(seqs, generator=g, device="cuda") * far).long() + 1
        else:  # the first half of the sequences holds pages, as many as half the pool has
            held = torch.zeros(seqs, dtype=torch.int64, device="cuda")
            n = seqs - case["count"] if kind == "fork" else seqs
            most = min(far, max(1, case["pool"] * page // (2 * n) - page))
            held[:n] = (torch.rand(n, generator=g, device="cuda") * most).long() + 1
        table = _table(g, held, page, case["pool"])
        s["table"] = torch.full((seqs, case["most"]), -1, dtype=torch.int32, device="cuda")
        s["table"][:, : table.shape[1]] = table
        s["lens"] = held.int()
        s["refs"] = torch.zeros(case["pool"], dtype=torch.int32, device="cuda")
        s["refs"][table[table >= 0].long()] = 1
        if kind == "reserve":
            pick = torch.randperm(seqs, generator=g, device="cuda")[: case["count"]]
            s["seq_ids"] = pick.int()
            s["new_lens"] = ((torch.rand(case["count"], generator=g, device="cuda") * far).long() + 1).int()
        else:
            s["pages"] = torch.empty(case["layers"], case["pool"], page, case["dim"], dtype=dt,
                                     device="cuda").normal_(generator=g)
        if kind == "fork":
            parents = min(4, n)
            s["children"] = torch.arange(n, seqs, device="cuda", dtype=torch.int32)
            s["parents"] = torch.randint(0, parents, (case["count"],), generator=g, device="cuda").int()
        if kind == "compact":
            s["kept"] = (s["table"].clone(), s["refs"].clone())
    else:
        lens = _lengths(g, case["rows"], case["far"], case["even"])
        pool = int(((lens + case["page"] - 1) // case["page"]).sum()) + 3
        s["table"] = _table(g, lens, case["page"], pool)
        s["pages"] = torch.empty(pool, case["page"], case["dim"], dtype=dt, device="cuda").normal_(generator=g)
        s["q"] = (2 * rand(case["rows"], case["heads"], case["dim"])).to(dt)
        s["seq_ids"] = torch.arange(case["rows"], device="cuda", dtype=torch.int32)
        s["positions"] = (lens - 1).int()
        s["sink"] = rand(case["heads"]) if case["sink"] else None
        s["longest"] = int(lens.max())
        s["scale"] = case["dim"] ** -0.5
    return s


# --------------------------------------------------------------------------------------------- plain forms
def _rotate(x, positions, freqs, offset, interleaved):
    """x [..., dim] in 32 bits, positions [...] of the same leading shape: the rotated copy."""
    angle = positions.double()[..., None] * freqs
    angle = angle - torch.round(angle / (2 * math.pi)) * (2 * math.pi)
    cos, sin = torch.cos(angle.float()), torch.sin(angle.float())
    rot = 2 * freqs.numel()
    part = x[..., offset:offset + rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rot // 2], part[..., rot // 2:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    both = torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)
    return torch.cat((x[..., :offset], both, x[..., offset + rot:]), -1)


def _plain_rotary(s):
    c = s["case"]
    x = s["x"].float()
    y = _rotate(x, s["positions"][..., None].expand(x.shape[:-1]), s["freqs"], s["offset"], c["interleaved"])
    return y.to(s["x"].dtype)


def _plain_append(s):
    c = s["case"]
    rows = _rotate(s["rows"].float(), s["positions"], s["freqs"], c["dim"] - c["rot"], c["interleaved"])
    seq, pos = s["seq_ids"].long(), s["positions"].long()
    s["pages"][s["table"][seq, pos // c["page"]].long(), pos % c["page"]] = rows.to(s["rows"].dtype)
    return s["pages"]


def _plain_free(s, seqs):
    seqs = seqs.long()
    held = s["table"][seqs]
    used = (held >= 0).int()
    s["refs"].scatter_add_(0, held.clamp(min=0).flatten().long(), -used.flatten())
    s["table"][seqs] = -1
    s["lens"][seqs] = 0


def _free_list(refs):
    """The pages without a holder, lowest first, in front of the others."""
    return torch.sort((refs > 0).to(torch.uint8), stable=True).indices.int()


def _plain_reserve(s, seqs, new_lens):
    page, seqs = s["case"]["page"], seqs.long()
    have = (s["lens"][seqs] + page - 1) // page
    want = torch.maximum((new_lens + page - 1) // page, have)
    need = want - have
    start = (need.cumsum(0) - need)[:, None]
    slot = torch.arange(s["table"].shape[1], device="cuda")[None]
    fresh = (slot >= have[:, None]) & (slot < want[:, None])
    at = (start + slot - have[:, None]).clamp(0, s["refs"].numel() - 1)
    got = torch.where(fresh, _free_list(s["refs"])[at], s["table"][seqs])
    s["table"][seqs] = got
    s["refs"].scatter_add_(0, got.clamp(min=0).flatten().long(), fresh.int().flatten())
    s["lens"][seqs] = torch.maximum(s["lens"][seqs], new_lens)


def _plain_fork(s, parents, children):
    page, parents, children = s["case"]["page"], parents.long(), children.long()
    lens = s["lens"][parents]
    full, rest = lens // page, lens % page
    slot = torch.arange(s["table"].shape[1], device="cuda")[None]
    rank = (rest > 0).int().cumsum(0) - (rest > 0).int()
    fresh = _free_list(s["refs"])[rank]
    held = s["table"][parents]
    row = torch.where(slot < full[:, None], held, -1)
    row = torch.where((slot == full[:, None]) & (rest > 0)[:, None], fresh[:, None], row)
    s["table"][children] = row
    s["refs"].scatter_add_(0, row.clamp(min=0).flatten().long(), (row >= 0).int().flatten())
    s["lens"][children] = lens
    some = rest > 0
    src = held.gather(1, full[:, None].clamp(max=held.shape[1] - 1).long())[some, 0].long()
    dst = fresh[some].long()
    mask = (torch.arange(page, device="cuda")[None] < rest[some][:, None])[None, :, :, None]
    s["pages"][:, dst] = torch.where(mask, s["pages"][:, src], s["pages"][:, dst])


def _plain_compact(s):
    refs = s["refs"]
    used = refs > 0
    n = used.sum()
    index = torch.arange(refs.numel(), device="cuda")
    hole, mover = ~used & (index < n), used & (index >= n)
    to = torch.sort((~hole).to(torch.uint8), stable=True).indices      # the k-th hole, for the k-th mover
    rank = mover.long().cumsum(0) - 1
    page_map = torch.where(used, torch.where(mover, to[rank.clamp(min=0)], index), -1)
    src = index[mover]
    dst = page_map[mover]
    s["pages"][:, dst] = s["pages"][:, src]
    moved = torch.zeros_like(refs)
    moved[page_map[used]] = refs[used]
    refs.copy_(moved)
    s["table"].copy_(torch.where(s["table"] >= 0, page_map[s["table"].clamp(min=0).long()].int(), -1))
    return page_map.int()


def _plain_attend(s):
    c = s["case"]
    page, pos = c["page"], s["positions"].long()[:, None]
    if c["window"]:  # the first tokens, then the window, of which the part before them or before the start is unseen
        first = torch.arange(min(c["first"], s["longest"]), device="cuda").expand(pos.shape[0], -1)
        key = torch.cat((first, pos + torch.arange(1 - c["window"], 1, device="cuda")), 1)
        seen = (key <= pos) & (key >= 0)
        seen[:, first.shape[1]:] &= key[:, first.shape[1]:] >= c["first"]
    else:
        key = torch.arange(s["longest"], device="cuda").expand(pos.shape[0], -1)
        seen = key <= pos
    key = torch.where(seen, key, 0)
    where = s["table"][s["seq_ids"].long()].long().gather(1, key // page) * page + key % page
    kv = s["pages"].view(-1, c["dim"])[where].float()                        # [T, keys, dim]
    kv = torch.where(seen[..., None], kv, 0.0)
    z = torch.matmul(s["q"].float(), kv.transpose(1, 2)) * s["scale"]
    z = z.masked_fill(~seen[:, None], float("-inf"))
    m = z.amax(-1, keepdim=True)
    if s["sink"] is not None:
        m = torch.maximum(m, s["sink"][None, :, None])
    p = torch.exp(z - m)
    den = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        den = den + torch.exp(s["sink"][None, :, None] - m)
    return torch.matmul(p / den, kv).to(s["q"].dtype)


# ----------------------------------------------------------------------------------------------------- run
def run(state):
    s, c = state, state["case"]
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(1, PACKAGE)
        from spark_b200 import kv_cache, rotary
    if c["op"] == "rotary":
        if own:
            y = rotary.rotary(s["x"], s["positions"], s["freqs"], interleaved=c["interleaved"], offset=s["offset"])
        else:
            y = _plain_rotary(s)
        if not c["train"]:
            return y
        return {"y": y.detach(), "grad": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    if c["op"] == "append":
        if not own:
            return _plain_append(s)
        kv_cache.append(s["pages"], s["rows"], s["table"], s["seq_ids"], s["positions"], s["freqs"],
                        interleaved=c["interleaved"])
        return s["pages"]
    if c["op"] == "pages":
        if c["kind"] == "reserve":
            if own:
                kv_cache.free(s["table"], s["lens"], s["refs"], s["seq_ids"])
                kv_cache.reserve(s["table"], s["lens"], s["refs"], s["seq_ids"], s["new_lens"], c["page"])
            else:
                _plain_free(s, s["seq_ids"])
                _plain_reserve(s, s["seq_ids"], s["new_lens"])
            return {"table": s["table"], "lens": s["lens"], "refs": s["refs"]}
        if c["kind"] == "fork":
            if own:
                kv_cache.free(s["table"], s["lens"], s["refs"], s["children"])
                kv_cache.fork(s["pages"], s["table"], s["lens"], s["refs"], s["parents"], s["children"])
            else:
                _plain_free(s, s["children"])
                _plain_fork(s, s["parents"], s["children"])
            return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "pages": s["pages"]}
        # the scheduler's tables, put back as they were before the pool was moved together
        s["table"].copy_(s["kept"][0])
        s["refs"].copy_(s["kept"][1])
        page_map = kv_cache.compact(s["pages"], s["table"], s["refs"]) if own else _plain_compact(s)
        return {"table": s["table"], "refs": s["refs"], "map": page_map, "pages": s["pages"]}
    if not own:
        return _plain_attend(s)
    return kv_cache.paged_attn(s["q"], s["pages"], s["table"], s["seq_ids"], s["positions"], s["sink"], s["scale"],
                               window=c["window"], first=c["first"])


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "rotary":
        n = c["batch"] * c["seq"] * c["heads"]
        passes = 2 if c["train"] else 1
        return {"bytes": passes * 2 * n * c["dim"] * size, "flops": passes * 3 * n * c["rot"]}
    if c["op"] == "append":
        return {"bytes": 2 * c["rows"] * c["dim"] * size + 8 * c["rows"], "flops": 3 * c["rows"] * c["rot"]}
    if c["op"] == "pages":
        # a sequence holds half of what it may on average; every table entry and count is touched once
        page_bytes = c["layers"] * c["page"] * c["dim"] * size
        tables = 8 * c["seqs"] * c["most"] + 8 * c["pool"]
        if c["kind"] == "reserve":
            return {"bytes": tables, "flops": 0}
        if c["kind"] == "fork":  # half of a last page for each child
            return {"bytes": tables + c["count"] * page_bytes, "flops": 0}
        # a quarter of the pool in use, of which three quarters lie behind its new end
        most = min(c["most"] * c["page"], max(1, c["pool"] * c["page"] // (2 * c["seqs"]) - c["page"]))
        held = c["seqs"] * (most / 2 / c["page"] + 0.5)
        return {"bytes": int(tables + 2 * held * (1 - held / c["pool"]) * page_bytes), "flops": 0}
    span = c["far"] if c["even"] else max(1.0, 0.55 * c["far"])
    if c["window"]:
        span = min(span, c["window"] + c["first"])
    pairs = c["rows"] * span
    return {"bytes": int(pairs * c["dim"] * size + 2 * c["rows"] * c["heads"] * c["dim"] * size),
            "flops": int(4 * pairs * c["heads"] * c["dim"])}


# --------------------------------------------------------------------------------------------------- exact
def _turned(x, pos, freqs, offset, interleaved, sign):
    """x [n, dim] and pos [n] in 64 bits as products of complex numbers."""
    rot = 2 * freqs.numel()
    y = x.clone()
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), sign * pos.double()[:, None] * freqs[None])
    if interleaved:
        first = torch.arange(offset, offset + rot, 2, device=x.device)
        second = first + 1
    else:
        first = torch.arange(offset, offset + rot // 2, device=x.device)
        second = first + rot // 2
    z = torch.complex(x[:, first], x[:, second]) * phase
    y[:, first], y[:, second] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":
        pos = s["positions"][..., None].expand(s["x"].shape[:-1]).reshape(-1)

        def turned(t, sign):
            flat = t.detach().double().reshape(-1, c["dim"])
            return _turned(flat, pos, s["freqs"], s["offset"], c["interleaved"], sign).reshape(t.shape)

        y = turned(s["x"], 1.0)
        return {"y": y, "grad": turned(s["grad"], -1.0)} if c["train"] else y
    if c["op"] == "append":
        out = s["pages"].double()
        rows = _turned(s["rows"].double(), s["positions"], s["freqs"], c["dim"] - c["rot"], c["interleaved"], 1.0)
        flat = out.view(-1, c["dim"])
        pos = s["positions"].long()
        flat[s["table"].long()[s["seq_ids"].long(), pos // c["page"]] * c["page"] + pos % c["page"]] = rows
        return out
    if c["op"] == "pages":
        return _exact_pages(c, s)
    out = torch.zeros(c["rows"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    table, position = s["table"].cpu(), s["positions"].cpu()
    for t in range(c["rows"]):
        p = int(position[t])
        keys = torch.arange(p + 1, device="cuda")
        if c["window"]:
            keys = torch.cat((keys[: min(c["first"], p + 1)], keys[max(min(c["first"], p + 1), p + 1 - c["window"]):]))
        where = table[t].cuda().long()[keys // c["page"]] * c["page"] + keys % c["page"]
        kv = s["pages"].view(-1, c["dim"])[where].double()
        z = (kv @ s["q"][t].double().T) * s["scale"]                     # [keys, heads]
        if s["sink"] is not None:
            z = torch.cat((z, s["sink"].double()[None]))
        p = torch.softmax(z, 0)[: kv.shape[0]]
        out[t] = p.T @ kv
    return out


def _exact_pages(c, s):
    """The page operations on lists, one sequence after the other."""
    page = c["page"]
    table, refs = s["table"].cpu().tolist(), s["refs"].cpu().tolist()
    lens = s["lens"].cpu().tolist()

    def lowest():
        p = refs.index(0)
        refs[p] = 1
        return p

    def drop(q):
        for p in table[q]:
            if p >= 0:
                refs[p] -= 1
        table[q] = [-1] * len(table[q])
        lens[q] = 0

    def tensors(**more):
        return {"table": torch.tensor(table, dtype=torch.int32), **more, "refs": torch.tensor(refs, dtype=torch.int32)}

    if c["kind"] == "reserve":
        for q in s["seq_ids"].tolist():
            drop(q)
        for q, n in zip(s["seq_ids"].tolist(), s["new_lens"].tolist()):
            for j in range((n + page - 1) // page):
                table[q][j] = lowest()
            lens[q] = n
        return tensors(lens=torch.tensor(lens, dtype=torch.int32))
    pages = s["pages"]
    if c["kind"] == "fork":
        for q in s["children"].tolist():
            drop(q)
        for a, b in zip(s["parents"].tolist(), s["children"].tolist()):
            lens[b] = lens[a]
            for j in range(lens[a] // page):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            rest = lens[a] % page
            if rest:
                p = lowest()
                table[b][lens[a] // page] = p
                pages[:, p, :rest] = pages[:, table[a][lens[a] // page], :rest]
        return tensors(lens=torch.tensor(lens, dtype=torch.int32)) | {"pages": pages.double()}
    used = [p for p, r in enumerate(refs) if r]
    holes = iter([p for p in range(len(used)) if not refs[p]])
    to = {p: (p if p < len(used) else next(holes)) for p in used}
    for p, q in to.items():
        if p != q:
            pages[:, q] = pages[:, p]
            refs[q], refs[p] = refs[p], 0
    table = [[to[p] if p >= 0 else -1 for p in row] for row in table]
    mapped = torch.tensor([to.get(p, -1) for p in range(c["pool"])], dtype=torch.int32)
    return tensors() | {"map": mapped, "pages": pages.double()}
