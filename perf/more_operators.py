"""Many continuations of one prompt: tables on the GPU, attention behind a shared prefix, log probabilities, as cases to time and compare.

A serving program that asks one prompt for many continuations (samples, candidates to be scored, drafts to be checked) holds the prompt's keys
once and lets every sequence's block table begin with the prompt's pages.

``tables``    the sequences' lengths change on the GPU (they grow by rows, are cut back or end): pages are taken from a stack of free ones or
              put back on it, and the step's block tables, first rows, positions, segments and slots are made; then the step is taken back
``shared``    causal attention of the rows of several sequences, in groups that share their first keys; the sequences of a group name the
              same pages there (a page that the prefix ends in is each sequence's own copy)
``logprobs``  of each row of logits the log probability of a given token and its rank, the row's entropy, and the alternatives with the
              largest logits (equal ones: the lowest index)

Lengths run evenly from the first to the last sequence or group of a case.
"""
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _shared(name, H, G, hd, groups, seqs, prefix, behind, rows=(1, 1), dtype="bfloat16", page=64):
    return {"name": name, "op": "shared", "dtype": dtype, "H": H, "G": G, "hd": hd, "page": page, "groups": groups, "seqs": seqs,
            "prefix_lo": prefix[0], "prefix_hi": prefix[1], "own_lo": behind[0], "own_hi": behind[1], "rows_lo": rows[0], "rows_hi": rows[1]}


def listed():
    return [
        # a decode step of a full small batch, every sequence one token further and one page in 64 new, and the step taken back
        {"name": "tables-64", "op": "tables", "seqs": 64, "page": 64, "len_lo": 1, "len_hi": 4096, "grow_hi": 1, "back": 0.0, "cap": 64},
        # very many sequences: portions of up to 60 tokens come in, a tenth of them lose their last tokens or end
        {"name": "tables-2000", "op": "tables", "seqs": 2000, "page": 16, "len_lo": 0, "len_hi": 9000, "grow_hi": 60, "back": 0.1, "cap": 65535},
        # eight samples of a prompt at the LFM2-1.2B shape, just begun: latency
        _shared("shared-8x2k", 32, 8, 64, 1, 8, (2048, 2048), (1, 150)),
        # a batch of samples of one prompt of 8,000 tokens
        _shared("shared-64x8k", 32, 8, 64, 1, 64, (8000, 8000), (1, 500)),
        # the same with heads of 128, more of them and longer continuations
        _shared("shared-256x4k", 32, 8, 128, 1, 256, (4096, 4096), (100, 700)),
        # questions about one very long text at the LFM2-350M shape
        _shared("shared-24x120k", 16, 8, 64, 1, 24, (120001, 120001), (5, 900)),
        # sixteen samples each of five prompts of different lengths, a few drafted tokens a step, small pages
        _shared("shared-5x16-drafts", 16, 4, 128, 5, 16, (701, 12000), (4, 300), (1, 4), page=16),
        # 32-bit, odd sizes
        _shared("shared-3x5-f32", 12, 4, 96, 3, 5, (333, 3001), (1, 200), (1, 2), dtype="float32", page=32),
        # the token a single request just got, with five alternatives
        {"name": "logprobs-1", "op": "logprobs", "dtype": "float32", "rows": 1, "vocab": 65536, "top": 5},
        # a full batch's tokens, twenty alternatives each
        {"name": "logprobs-64", "op": "logprobs", "dtype": "float32", "rows": 64, "vocab": 65536, "top": 20},
        # a prompt's portion is scored, no alternatives
        {"name": "logprobs-2048", "op": "logprobs", "dtype": "float32", "rows": 2048, "vocab": 65536, "top": 0},
        # 16-bit logits of an odd vocabulary, whose rows start at any address
        {"name": "logprobs-300-bf16", "op": "logprobs", "dtype": "bfloat16", "rows": 300, "vocab": 100003, "top": 32},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["tables", "shared", "shared", "shared", "logprobs", "logprobs"])
    if op == "tables":
        seqs, cap = _log(rng, 1, 2000), 65535
        hi = rng.choice([1, 1, 4, max(1, min(2000, 60000 // seqs))])
        return {"op": op, "seqs": seqs, "page": rng.choice([1, 16, 32, 64, 100, 128]), "len_lo": rng.randint(0, 20), "len_hi": _log(rng, 30, 9000), "grow_hi": hi,
                "back": rng.choice([0.0, 0.1, 0.5]), "cap": min(cap, seqs * hi + rng.randint(0, 50))}
    if op == "logprobs":
        vocab = _log(rng, 500, 260000)
        rows = _log(rng, 1, max(2, min(2048, 130000000 // vocab)))
        return {"op": op, "dtype": rng.choice(["float32", "float32", "bfloat16"]), "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)])}
    G, per, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8, 12]), rng.choice([32, 64, 64, 64, 96, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    groups = rng.choice([1, 1, 1, 2, _log(rng, 2, 8)])
    seqs = _log(rng, 2, max(2, min(256, 1024 * 16 // (groups * G * per))))
    rows = (1, rng.choice([1, 1, 1, 2, 4]))
    keys = 24000000 // (G * hd * groups * (2 if dtype == "float32" else 1))                  # of a prefix, at most
    prefix = _log(rng, 16, max(32, min(100000, keys, 400000000 // (G * per * groups * seqs * rows[1]))))
    own_hi = _log(rng, rows[1], max(8, min(900, keys * groups // (groups * seqs))))
    c = _shared("", G * per, G, hd, groups, seqs, (rng.randint(prefix // 2, prefix), prefix), (rng.randint(rows[1], own_hi), own_hi), rows, dtype,
                rng.choice([16, 32, 64, 128]))
    c.pop("name")
    return c


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * seed + 29)
    st = {"case": c}
    return {"tables": _prepare_tables, "shared": _prepare_shared, "logprobs": _prepare_logprobs}[c["op"]](c, gen, st)


def _prepare_tables(c, gen, st):
    S, ps, cap = c["seqs"], c["page"], c["cap"]
    rand = lambda hi: torch.randint(0, hi + 1, (S,), generator=gen, device="cuda")  # noqa: E731
    seq = torch.arange(S, device="cuda")
    length = c["len_lo"] + rand(c["len_hi"] - c["len_lo"])
    length = torch.where(seq % 8 == 5, rand(2 * ps).clamp(max=c["len_hi"]), length)
    grow = rand(c["grow_hi"] - 1) + 1
    if S * c["grow_hi"] > cap:                                                     # (no more rows than there is room for)
        grow = grow * cap // (S * c["grow_hi"])
    back = torch.minimum(rand(min(3 * ps, cap // S) - 1) + 1, length)              # short sequences end, others lose their last tokens
    cut = (torch.rand(S, generator=gen, device="cuda") < c["back"]) & (back > 0)
    delta = torch.where(cut, -back, grow)
    after = length + delta
    # the first blocks of every other sequence are a shared prompt's
    own_from = torch.where(seq % 2 == 0, torch.zeros_like(length), torch.minimum(length, after) // ps // 2)
    blocks = (length + ps - 1) // ps
    width, held = -(-(c["len_hi"] + c["grow_hi"]) // ps) + 1, int(blocks.sum())
    P = S * (-(-c["len_hi"] // ps) + -(-c["grow_hi"] // ps) + 2)
    order = torch.randperm(P, generator=gen, device="cuda").to(torch.int32)
    st["table"] = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    st["table"][torch.arange(width, device="cuda")[None] < blocks[:, None]] = order[:held]
    st["free"] = torch.zeros(P, dtype=torch.int32, device="cuda")
    st["free"][:P - held] = order[held:]
    st["n_free"] = torch.tensor([P - held], dtype=torch.int32, device="cuda")
    st["length"], st["own_from"] = length.to(torch.int32), own_from.to(torch.int32)
    st["deltas"] = [delta.to(torch.int32), (-delta).to(torch.int32)]
    new = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    st["steps"] = [{"cu_rows": new(S + 1), "seg_pos": new(S), "row_seg": new(cap), "positions": new(cap), "slots": new(cap), "status": new(1)}
                   for _ in range(2)]
    return st


def _prepare_shared(c, gen, st):
    H, G, hd, ps, dt = c["H"], c["G"], c["hd"], c["page"], DTYPES[c["dtype"]]
    prefix = _spread(c["prefix_lo"], c["prefix_hi"], c["groups"])
    n_seq = c["groups"] * c["seqs"]
    behind, rows = _spread(c["own_lo"], c["own_hi"], n_seq), _spread(c["rows_lo"], c["rows_hi"], n_seq)
    P = [prefix[i // c["seqs"]] for i in range(n_seq)]
    total = [p + o for p, o in zip(P, behind)]
    width = max(-(-t // ps) for t in total)
    whole = [p // ps for p in prefix]
    need = sum(whole) + sum(-(-t // ps) - p // ps for t, p in zip(total, P))
    order = torch.randperm(need + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((n_seq, width), dtype=torch.int32, device="cuda")
    at, cache = 0, torch.empty((need + 3, 2, G, ps, hd), dtype=dt, device="cuda")
    # keys and values as they are: some channels of a head are much larger than the others, and shifted
    big = 1.0 + 4.0 * (torch.rand((2, G, 1, hd), generator=gen, device="cuda") < 0.05)
    shift = 0.3 * torch.randn((2, G, 1, hd), generator=gen, device="cuda")
    step = max(1, (1 << 25) // (2 * G * ps * hd))
    for a in range(0, need + 3, step):
        b = min(need + 3, a + step)
        cache[a:b] = ((torch.randn((b - a, 2, G, ps, hd), generator=gen, device="cuda") + shift) * big).to(dt)
    for g in range(c["groups"]):
        table[g * c["seqs"]:(g + 1) * c["seqs"], :whole[g]] = order[at:at + whole[g]]
        at += whole[g]
    tails = []
    for i in range(n_seq):
        w, n = whole[i // c["seqs"]], -(-total[i] // ps)
        table[i, w:n] = order[at:at + n - w]
        at += n - w
        tails.append(P[i] % ps)
    # a page that a prefix ends in: every sequence's copy holds the same first keys
    for g in range(c["groups"]):
        t = prefix[g] % ps
        if t:
            mine = table[g * c["seqs"]:(g + 1) * c["seqs"], whole[g]].long()
            cache[mine[1:], :, :, :t] = cache[mine[0], :, :, :t]
    st["cache"], st["table"] = cache, table
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    st["q"] = torch.randn((cu[-1], H * hd), generator=gen, device="cuda").to(dt)
    st["cu_rows"], st["seg_pos"] = i32(cu), i32([t - r for t, r in zip(total, rows)])
    st["group_seqs"], st["prefix_len"] = i32([g * c["seqs"] for g in range(c["groups"] + 1)]), i32(prefix)
    st["host"] = {"prefix": prefix, "own": behind, "rows": rows, "cu": cu}
    st["max_rows"], st["max_prefix"], st["max_own"] = max(rows), max(prefix), max(behind)
    st["max_group_rows"] = max(cu[(g + 1) * c["seqs"]] - cu[g * c["seqs"]] for g in range(c["groups"]))
    st["out"] = torch.empty_like(st["q"])
    return st


def _prepare_logprobs(c, gen, st):
    n, V = c["rows"], c["vocab"]
    x = torch.randn((n, V), generator=gen, device="cuda", dtype=torch.float32)
    x.mul_(2.5)
    for r in range(0, n, 256):                                                     # some rows are sure of a few tokens
        part = x[r:r + 256]
        sure = torch.randint(0, V, (part.shape[0], 3), generator=gen, device="cuda")
        part.scatter_add_(1, sure, 12.0 * torch.rand((part.shape[0], 3), generator=gen, device="cuda"))
    if V > 64:
        x[:, V - 40:] = float("-inf")                                              # places of the vocabulary that no token has
    st["logits"] = x.to(DTYPES[c["dtype"]])
    ids = torch.randint(0, V - 40 if V > 64 else V, (n,), generator=gen, device="cuda")
    likely = torch.rand(n, generator=gen, device="cuda") < 0.5
    st["ids"] = torch.where(likely, st["logits"].float().argmax(1), ids).to(torch.int32)
    if n > 4:
        st["ids"][n // 2] = -1                                                     # a row that asks for no token
    return st


# ------------------------------------------------------------------------------------------------ one pass

def run(st):
    return (_own if own else {"tables": _plain_tables, "shared": _plain_shared, "logprobs": _plain_logprobs}[st["case"]["op"]])(st)


def _tables_out(st):
    return [st["table"], st["length"], st["free"], st["n_free"]] + [list(o.values()) for o in st["steps"]]


def _own(st):
    c = st["case"]
    if c["op"] == "tables":
        from kappai_b200.ops.tables import page_tables

        # a step, and the step that takes it back (every draft was refused): the pages lie on the stack as they did
        for delta, o in zip(st["deltas"], st["steps"]):
            page_tables(st["table"], st["length"], delta, st["free"], st["n_free"], c["page"], o["cu_rows"], o["seg_pos"], o["row_seg"],
                        o["positions"], o["slots"], o["status"], own_from=st["own_from"])
        return _tables_out(st)
    if c["op"] == "shared":
        from kappai_b200.ops.shared import attention_shared

        attention_shared(st["q"], st["cache"], st["table"], st["cu_rows"], st["seg_pos"], st["group_seqs"], st["prefix_len"], st["out"], c["hd"] ** -0.5,
                         c["page"], c["H"], c["G"], c["hd"], st["max_rows"], st["max_group_rows"], st["max_prefix"], st["max_own"])
        return (st["out"],)
    from kappai_b200.ops.logprobs import token_logprobs

    got = token_logprobs(st["logits"], st["ids"], c["top"])
    return got.logprob, got.entropy, got.rank, got.top_ids, got.top_logprobs


def _plain_tables(st):
    for delta, o in zip(st["deltas"], st["steps"]):
        _plain_step(st, delta, o)
    return _tables_out(st)


def _plain_step(st, delta, o):
    c = st["case"]
    ps, S, cap = c["page"], c["seqs"], c["cap"]
    table, free = st["table"], st["free"]
    L, d, keep = st["length"].long(), delta.long(), st["own_from"].long()
    dev, W, P = L.device, table.shape[1], free.shape[0]
    blocks = (L + ps - 1) // ps
    keep = torch.minimum(keep, blocks)
    ended = L + d <= 0
    after = torch.where(ended, torch.zeros_like(L), torch.where(d < 0, torch.minimum(L, torch.maximum(L + d, keep * ps)), L + d))
    blocks_after = (after + ps - 1) // ps
    rows = d.clamp(min=0)
    n_free = st["n_free"].long()
    back_from = torch.where(blocks_after < blocks, torch.maximum(blocks_after, keep), blocks)
    back, taken = (blocks - back_from).clamp(min=0), (blocks_after - blocks).clamp(min=0)
    short, wide, many = taken.sum() > n_free + back.sum(), (blocks_after > W).any(), rows.sum() > cap
    status = short.long() + 2 * wide.long() + 4 * many.long()
    ok = status == 0
    rows, back, taken = rows * ok, back * ok, taken * ok
    cu = torch.nn.functional.pad(rows.cumsum(0), (1, 0))
    block = torch.arange(W, device=dev)
    # pages that come back lie on top of the stack, the first sequence's first one uppermost
    returned = (block >= back_from[:, None]) & (block < (back_from + back)[:, None])
    top = n_free + back.sum()
    place = top - 1 - ((back.cumsum(0) - back)[:, None] + block - back_from[:, None])
    stack = torch.nn.functional.pad(free, (0, 1))                                  # (one more place, for what is not pushed)
    stack.scatter_(0, torch.where(returned, place, torch.full_like(place, P)).flatten(), table.flatten())
    gone = (block >= torch.where(ended, torch.zeros_like(L), back_from)[:, None]) & (block < blocks[:, None]) & (blocks_after < blocks)[:, None] & ok
    table.masked_fill_(gone, -1)
    # the first sequence's first new page is the uppermost
    fresh = (block >= blocks[:, None]) & (block < (blocks + taken)[:, None])
    which = top - 1 - ((taken.cumsum(0) - taken)[:, None] + block - blocks[:, None])
    table.copy_(torch.where(fresh, stack[which.clamp(0, P - 1)], table))
    free.copy_(stack[:P])
    st["n_free"].copy_(top - taken.sum())
    st["length"].copy_(torch.where(ok, after, L))
    o["cu_rows"].copy_(cu)
    o["seg_pos"].copy_(torch.where(ok & (d < 0), after, L))
    r = torch.arange(cap, device=dev)
    live = r < cu[-1]
    seg = torch.searchsorted(cu[1:].contiguous(), r, right=True).clamp(max=S - 1)
    pos = L[seg] + r - cu[seg]
    page = table[seg, (pos // ps).clamp(0, W - 1)].long()
    o["row_seg"].copy_(torch.where(live, seg, torch.zeros_like(seg)))
    o["positions"].copy_(torch.where(live, pos, torch.full_like(pos, -1)))
    o["slots"].copy_(torch.where(live, page * ps + pos % ps, torch.full_like(pos, -1)))
    o["status"].copy_(status)


def _plain_shared(st):
    c, host = st["case"], st["host"]
    H, G, hd, ps, dev = c["H"], c["G"], c["hd"], c["page"], st["q"].device
    n, B = st["q"].shape[0], c["seqs"]
    q = st["q"].float().unflatten(1, (G, H // G, hd)) * hd ** -0.5                 # [n, G, R, hd]
    cu, pos, table = st["cu_rows"].long(), st["seg_pos"].long(), st["table"].long()
    row = torch.arange(n, device=dev)
    seg = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    at = pos[seg] + row - cu[seg]
    plen = st["prefix_len"].long().repeat_interleave(B)[seg]
    tops, sums, outs = [], [], []
    # the group's keys: one product for all its rows
    s0, l0, o0 = (torch.empty(sh, device=dev) for sh in ((n, G, H // G, 1), (n, G, H // G, 1), (n, G, H // G, hd)))
    for g in range(c["groups"]):
        P, a, b = host["prefix"][g], host["cu"][g * B], host["cu"][(g + 1) * B]
        k, v = (st["cache"][table[g * B, :-(-P // ps)], w].transpose(0, 1).flatten(1, 2)[:, :P].float() for w in (0, 1))     # [G, P, hd]
        step = max(1, (1 << 27) // (P * H))
        for i in range(a, b, step):
            j = min(b, i + step)
            s = q[i:j].permute(1, 0, 2, 3).flatten(1, 2) @ k.transpose(1, 2)       # [G, rows R, P]
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            back = lambda t: t.unflatten(1, (j - i, H // G)).transpose(0, 1)  # noqa: E731
            s0[i:j], l0[i:j], o0[i:j] = back(top), back(p.sum(-1, keepdim=True)), back(p @ v)
    tops.append(s0), sums.append(l0), outs.append(o0)
    # the keys behind it, each sequence's by themselves, some rows at a time
    step = max(1, (1 << 26) // (st["max_own"] * G * hd))
    s1, l1, o1 = torch.empty_like(s0), torch.empty_like(l0), torch.empty_like(o0)
    for i in range(0, n, step):
        j = min(n, i + step)
        key = plen[i:j, None] + torch.arange(st["max_own"], device=dev)
        sees = key <= at[i:j, None]
        page = table[seg[i:j, None], (key // ps).clamp(max=table.shape[1] - 1)]
        k, v = (st["cache"][page, w, :, key % ps].float().masked_fill(~sees[..., None, None], 0.0) for w in (0, 1))          # [rows, keys, G, hd]
        s = (q[i:j] @ k.permute(0, 2, 3, 1)).masked_fill(~sees[:, None, None], float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        s1[i:j], l1[i:j], o1[i:j] = top, p.sum(-1, keepdim=True), p @ v.transpose(1, 2)
    top = torch.maximum(s0, s1)
    a, b = torch.exp(s0 - top), torch.exp(s1 - top)
    st["out"].copy_(((a * o0 + b * o1) / (a * l0 + b * l1)).flatten(1))
    return (st["out"],)


def _plain_logprobs(st):
    c = st["case"]
    x, ids, k = st["logits"], st["ids"].long(), c["top"]
    parts = []
    for a in range(0, x.shape[0], 512):
        f, i = x[a:a + 512].float(), ids[a:a + 512]
        top = f.amax(1, keepdim=True)
        e = torch.exp(f - top)
        total = e.sum(1, keepdim=True)
        lse = top + torch.log(total)
        p = e / total
        entropy = torch.log(total)[:, 0] - torch.where(p > 0, p * (f - top), torch.zeros_like(p)).sum(1)
        there = i >= 0
        mine = f.gather(1, i.clamp(min=0)[:, None])
        lp = torch.where(there, (mine - lse)[:, 0], torch.zeros_like(entropy))
        rank = torch.where(there, (f > mine).sum(1), torch.full_like(i, -1)).to(torch.int32)
        best = torch.sort(f, dim=1, descending=True, stable=True) if k else None
        tid = best.indices[:, :k].to(torch.int32) if k else torch.empty((f.shape[0], 0), dtype=torch.int32, device=f.device)
        tlp = best.values[:, :k] - lse if k else torch.empty((f.shape[0], 0), device=f.device)
        parts.append((lp, entropy, rank, tid, tlp))
    return tuple(torch.cat(t) for t in zip(*parts))


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(c):
    if c["op"] == "tables":                                                        # two steps: lengths, changes, first own blocks; lengths, first rows, positions
        S, cap = c["seqs"], c["cap"]
        pages = S * (1 + c["grow_hi"] // (2 * c["page"])) // 2
        return {"bytes": 2 * 4 * (6 * S + 3 * cap + 2 * pages + 4), "flops": 2 * (8 * S + 3 * cap)}
    if c["op"] == "logprobs":
        item = 2 if c["dtype"] == "bfloat16" else 4
        n, V = c["rows"], c["vocab"]
        return {"bytes": n * (V * item + 4 + 12 + 8 * c["top"]), "flops": 5 * n * V}
    H, G, hd, item = c["H"], c["G"], c["hd"], 2 if c["dtype"] == "bfloat16" else 4
    prefix = _spread(c["prefix_lo"], c["prefix_hi"], c["groups"])
    n_seq = c["groups"] * c["seqs"]
    behind, rows = _spread(c["own_lo"], c["own_hi"], n_seq), _spread(c["rows_lo"], c["rows_hi"], n_seq)
    pairs = sum(r * (prefix[i // c["seqs"]] + o) - r * (r - 1) // 2 for i, (o, r) in enumerate(zip(behind, rows)))
    return {"bytes": (sum(prefix) + sum(behind)) * 2 * G * hd * item + 2 * sum(rows) * H * hd * item, "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "tables":
        return None                                                                # whole numbers: the plain form's are compared
    if c["op"] == "logprobs":
        lps, ents, tlps = [], [], []
        for r in range(0, c["rows"], 128):
            x = st["logits"][r:r + 128].double()
            lse = torch.logsumexp(x, 1)
            lp = x - lse[:, None]
            p = lp.exp()
            ents.append(-(p * lp.masked_fill(p == 0, 0.0)).sum(1))
            ids = st["ids"][r:r + 128].long()
            lps.append(torch.where(ids >= 0, lp[torch.arange(len(ids), device="cuda"), ids.clamp(min=0)], torch.zeros_like(lse)))
            tlps.append(torch.topk(lp, c["top"], 1).values)
        return [torch.cat(lps), torch.cat(ents), None, None, torch.cat(tlps)]
    H, G, hd, ps = c["H"], c["G"], c["hd"], c["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda").unflatten(1, (G, H // G, hd))
    q, cu, first = st["q"].double().unflatten(1, (G, H // G, hd)), st["host"]["cu"], st["seg_pos"].tolist()
    budget = 0
    for i in range(len(first)):
        n = first[i] + cu[i + 1] - cu[i]
        budget += n * G * hd
    if budget > 6e9:
        return None
    for i in range(len(first)):
        a, b = cu[i], cu[i + 1]
        n = first[i] + b - a
        key = torch.arange(n, device="cuda")
        pages = st["table"][i].long()[key // ps]
        last = first[i] + torch.arange(b - a, device="cuda")
        for g in range(G):
            k, v = st["cache"][pages, 0, g, key % ps].double(), st["cache"][pages, 1, g, key % ps].double()
            s = torch.einsum("rhd,kd->rhk", q[a:b, g], k) / hd ** 0.5
            s = torch.where(key <= last[:, None, None], s, torch.full_like(s, float("-inf")))
            out[a:b, g] = torch.einsum("rhk,kd->rhd", torch.softmax(s, -1), v)
    return [out.flatten(1)]
