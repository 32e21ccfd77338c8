"""Paged caches of sequences that share prefixes: what is measured of the calls that keep them.

Three operators that one step of a serving loop, or of sampling a group of answers to one prompt, runs one after the other:

  pages   block tables, slots and positions of the tokens that every request adds, from the requests' lengths and a stack of free pages
          (extend), and the pages of finished requests back onto that stack (release)
  store   new rows of a layer's fused q / k / v projection: per-head norms, rotation, keys and values into their slots, queries as 16-bit rows
  attn    attention of those rows over the pages of their own request, causal, and over the pages of a prefix that a group of requests shares

A pool holds keys (or values) as [n_pages][n_kv][page][hd]; page tables hold page numbers. Request r owns d_len[r] tokens and reads the prefix of
its group before them.
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
THETA = 1e6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# query heads, key / value heads and head dimension: those of this framework's Qwen3 and Gemma3 configurations, and smaller ones
HEADS = [(32, 8, 128), (16, 8, 128), (8, 2, 64), (4, 1, 256), (16, 2, 64), (8, 8, 128), (5, 1, 128)]


def listed():
    return [
        # one decode step of 32 sequences: every request adds a token
        dict(name="extend-step", op="extend", requests=32, page=16, longest=2000, most_new=1),
        # a full server between prompts: many requests, portions of all lengths
        dict(name="extend-portions", op="extend", requests=1000, page=16, longest=8000, most_new=201),
        # half of the requests of a long run are done
        dict(name="release", op="release", requests=700, page=32, longest=16000, most_new=1),
        # the rows of one decode step, Qwen3-4B's heads
        dict(name="store-step-f16", op="store", dtype="f16", rows=32, heads=32, kv=8, hd=128, page=16),
        # portions of prompts in one pass over the weights
        dict(name="store-portion-bf16", op="store", dtype="bf16", rows=8191, heads=16, kv=8, hd=128, page=16),
        # four chats behind a short system prompt: launches and latency
        dict(name="attn-chats-f16", op="attn", dtype="f16", heads=16, kv=8, hd=128, page=16, requests=4, groups=1, prefix=700, longest=60, most_new=1),
        # 32 answers to one long prompt, in mid-answer
        dict(name="attn-group-f16", op="attn", dtype="f16", heads=32, kv=8, hd=128, page=16, requests=32, groups=1, prefix=8199, longest=1024, most_new=1),
        # groups of several prompts, narrow heads
        dict(name="attn-groups-bf16", op="attn", dtype="bf16", heads=16, kv=2, hd=64, page=32, requests=128, groups=8, prefix=4000, longest=700, most_new=1),
        # wide heads, one key / value head
        dict(name="attn-wide-f16", op="attn", dtype="f16", heads=4, kv=1, hd=256, page=64, requests=24, groups=1, prefix=2000, longest=900, most_new=1),
        # a few drafted tokens a request, checked together
        dict(name="attn-drafts-f16", op="attn", dtype="f16", heads=32, kv=8, hd=128, page=16, requests=61, groups=2, prefix=16001, longest=1500, most_new=8),
        # portions of prompts that continue a shared beginning
        dict(name="attn-portions-bf16", op="attn", dtype="bf16", heads=32, kv=8, hd=128, page=64, requests=4, groups=1, prefix=4096, longest=1800, most_new=1024),
        # many answers about one book
        dict(name="attn-long-f16", op="attn", dtype="f16", heads=32, kv=8, hd=128, page=16, requests=64, groups=1, prefix=65521, longest=4096, most_new=1),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["extend", "release", "store", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    if op in ("extend", "release"):
        return dict(op=op, requests=_spread(rng, 1, 1024), page=page, longest=_spread(rng, 1, 16000), most_new=1 if op == "release" else _spread(rng, 1, 200))
    heads, kv, hd = rng.choice(HEADS)
    dtype = rng.choice(["f16", "bf16"])
    if op == "store":
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, 8191), heads=heads, kv=kv, hd=hd, page=page)
    most_new = _spread(rng, 1, 1024) if rng.random() < 0.3 else rng.choice([1, 1, 2, 5, 8])
    requests = _spread(rng, 1, 128 if most_new <= 8 else 4)
    groups = rng.choice([0, 1, 1, 1 + rng.randrange(requests)])
    case = dict(op=op, dtype=dtype, heads=heads, kv=kv, hd=hd, page=page, requests=requests, groups=groups, prefix=_spread(rng, 1, 32000) if groups <= 2 else _spread(rng, 1, 4000),
                longest=most_new + _spread(rng, 1, 2000 if requests > 16 else 8000), most_new=most_new)
    most = max(_cost(c) for c in listed())
    while _cost(case) > most:                                            # many new rows behind a long prefix
        case.update(prefix=case["prefix"] * 2 // 3, longest=max(most_new, case["longest"] * 2 // 3))
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ------------------------------------------------------------------ lengths: of the case alone, so that its work is known

def _lengths(case):
    """Tokens of every request with its new ones, new ones, first requests of the groups (and the end), and the groups' prefixes."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, most = case["requests"], case["most_new"]
    if case["op"] == "attn":
        new = [rng.randint(1, most) for _ in range(n)]
    else:
        new = [rng.randint(0, most) if most > 1 else 1 for _ in range(n)]
    total = [max(a, rng.randint(1, case["longest"])) for a in new]
    if case["op"] == "attn":
        total[0] = max(new[0], case["longest"])
    groups = case.get("groups", 0)
    cuts = sorted(rng.sample(range(1, n), groups - 1)) if groups > 1 else []
    prefix = [case["prefix"] if g == 0 else rng.randint(0, case["prefix"]) for g in range(groups)]
    return total, new, ([0] + cuts + [n] if groups else [0]), prefix


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] in ("extend", "release"):
        total, new, _, _ = _lengths(case)
        n, page = len(total), case["page"]
        if case["op"] == "extend":
            fresh = sum(_pages(t, page) - _pages(t - a, page) for t, a in zip(total, new))
            rows = sum(new)
            return {"bytes": 4 * (5 * n + 2 * rows + 2 * fresh), "flops": 0}
        done = sum(_pages(t, page) for i, t in enumerate(total) if i % 2 == 0)
        return {"bytes": 4 * (3 * n + 2 * done), "flops": 0}
    wide = (case["heads"] + 2 * case["kv"]) * case["hd"]
    if case["op"] == "store":
        return {"bytes": case["rows"] * (6 * wide + 8), "flops": case["rows"] * 8 * wide}
    total, new, starts, prefix = _lengths(case)
    rows, keys = sum(new), sum(total) + sum(prefix)
    seen = sum(a * (t - a) + a * (a + 1) // 2 for t, a in zip(total, new))
    for g, p in enumerate(prefix):
        seen += p * sum(new[starts[g]:starts[g + 1]])
    return {"bytes": 4 * keys * case["kv"] * case["hd"] + 4 * rows * case["heads"] * case["hd"], "flops": 4 * seen * case["heads"] * case["hd"]}


# ------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {k: v for k, v in case.items() if k != "name"}
    if case["op"] == "store":
        rows, page, hd = case["rows"], case["page"], case["hd"]
        n_pages = _pages(rows, page) + 3
        rng = random.Random(seed)
        first = rng.randrange(4000)                                   # a portion that starts anywhere, after others
        s["qkv"] = torch.randn(rows, (case["heads"] + 2 * case["kv"]) * hd, generator=gen, device="cuda")
        s["q_gamma"], s["k_gamma"] = (1 + 0.1 * torch.randn(hd, generator=gen, device="cuda") for _ in range(2))
        s["inv_freq"] = (THETA ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)).float()
        order = torch.randperm(n_pages, generator=gen, device="cuda")
        at = torch.arange(rows, device="cuda")
        s["slot"] = (order[at // page] * page + at % page).int()
        s["pos"] = (first + at).int()
        s["count"] = _ints([rows])
        s["k_pool"], s["v_pool"] = (torch.zeros(n_pages, case["kv"], page, hd, dtype=DTYPES[case["dtype"]], device="cuda") for _ in range(2))
        s["q"] = torch.zeros(rows, case["heads"] * hd, dtype=DTYPES[case["dtype"]], device="cuda")
        s["n_pages"] = n_pages
        return s
    total, new, starts, prefix = _lengths(case)
    page, n = case["page"], case["requests"]
    before = [t - a for t, a in zip(total, new)] if case["op"] == "extend" else total
    held, all_pages = [_pages(t, page) for t in before], sum(_pages(t, page) for t in total)
    if case["op"] != "attn":
        n_pages = all_pages + 5
        order = torch.randperm(n_pages, generator=gen, device="cuda").int()
        ld = max(_pages(t, page) for t in total) + 1
        table = torch.full((n, ld), -1, dtype=torch.int32, device="cuda")
        counts = _ints(held).long()
        here = torch.arange(ld, device="cuda") < counts[:, None]
        table[here] = order[:sum(held)]
        s.update(len=_ints(before), new=_ints(new if case["op"] == "extend" else [1 - i % 2 for i in range(n)]), base=_ints([7 * i for i in range(n)]), table=table,
                 free=torch.cat([order[sum(held):].flip(0), torch.full((sum(held),), -1, dtype=torch.int32, device="cuda")]), free_n=_ints([n_pages - sum(held)]),
                 len_out=torch.zeros(n, dtype=torch.int32, device="cuda"), free_n_out=_ints([0]), n_pages=n_pages, total_rows=sum(new),
                 row_start=torch.zeros(n + 1, dtype=torch.int32, device="cuda"), slot=torch.full((max(1, sum(new)),), -1, dtype=torch.int32, device="cuda"),
                 pos=torch.full((max(1, sum(new)),), -1, dtype=torch.int32, device="cuda"), status=_ints([0]))
        s["fresh"] = sum(_pages(t, page) for t in total) - sum(held)
        return s
    dtype, heads, kv, hd = DTYPES[case["dtype"]], case["heads"], case["kv"], case["hd"]
    p_pages = [_pages(p, page) for p in prefix]
    n_pages = sum(held) + sum(p_pages) + 1
    order = torch.randperm(n_pages, generator=gen, device="cuda").int()
    ld, p_ld = max(held), max(p_pages + [1])
    table, p_table = torch.zeros(n, ld, dtype=torch.int32, device="cuda"), torch.zeros(max(1, len(prefix)), p_ld, dtype=torch.int32, device="cuda")
    table[torch.arange(ld, device="cuda") < _ints(held).long()[:, None]] = order[:sum(held)]
    if prefix:
        p_table[torch.arange(p_ld, device="cuda") < _ints(p_pages).long()[:, None]] = order[sum(held):sum(held) + sum(p_pages)]
    rows = sum(new)
    s["k_pool"], s["v_pool"] = (torch.empty(n_pages, kv, page, hd, dtype=dtype, device="cuda").normal_(generator=gen) for _ in range(2))
    s["q"] = (2.5 * torch.randn(rows, heads * hd, generator=gen, device="cuda")).to(dtype)        # scores spread over a few units, as a model's are
    s["out"] = torch.zeros(rows, heads * hd, dtype=dtype, device="cuda")
    ends = [0]
    for a in new:
        ends.append(ends[-1] + a)
    # what the program knows on the host: bounds of its buffers
    s.update(n_pages=n_pages, rows=rows, longest_own=max(total), most=max(new), longest_prefix=max(prefix + [0]), most_group=max([ends[b] - ends[a] for a, b in zip(starts, starts[1:])] + [0]),
             table=table, p_table=p_table, len=_ints(total), row_start=_ints(ends), group_start=_ints(starts), prefix_len=_ints(prefix or [0]))
    return s


# ------------------------------------------------------------------ the plain forms

def _plain_extend(s):
    page, n, rows = s["page"], s["requests"], s["total_rows"]
    length, new = s["len"].long(), s["new"].long()
    held, wanted = (length + page - 1) // page, (length + new + page - 1) // page
    first_page, first_row = torch.cumsum(wanted - held, 0) - (wanted - held), torch.cumsum(new, 0) - new
    requests = torch.arange(n, device="cuda")
    owner = torch.repeat_interleave(requests, wanted - held, output_size=s["fresh"])
    at = torch.arange(s["fresh"], device="cuda")
    s["table"][owner, held[owner] + at - first_page[owner]] = s["free"][s["free_n"].long() - 1 - at]
    owner = torch.repeat_interleave(requests, new, output_size=rows)
    token = length[owner] + torch.arange(rows, device="cuda") - first_row[owner]
    s["slot"][:rows] = (s["table"][owner, token // page].long() * page + token % page).int()
    s["pos"][:rows] = (s["base"].long()[owner] + token).int()
    s["row_start"][0] = 0
    s["row_start"][1:] = torch.cumsum(new, 0).int()
    s["len_out"].copy_((length + new).int())
    s["free_n_out"].copy_((s["free_n"] - (wanted - held).sum()).int())


def _plain_release(s):
    page = s["page"]
    gone = s["new"] != 0
    pages = torch.where(gone, (s["len"].long() + page - 1) // page, 0)
    taken = torch.arange(s["table"].shape[1], device="cuda") < pages[:, None]
    back = s["table"][taken]
    s["free"][s["free_n"].long() + torch.arange(back.numel(), device="cuda")] = back
    s["free_n_out"].copy_((s["free_n"] + pages.sum()).int())
    s["len_out"].copy_(torch.where(gone, 0, s["len"]))


def _plain_store(s):
    heads, kv, hd, page = s["heads"], s["kv"], s["hd"], s["page"]
    x = s["qkv"].view(s["rows"], heads + 2 * kv, hd)
    gamma = torch.cat([s["q_gamma"].expand(heads, hd), s["k_gamma"].expand(kv, hd)])
    qk = x[:, :heads + kv]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * gamma
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()            # far positions: an angle in 32 bits is off by whole steps of the type
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    lo, hi = qk[..., :hd // 2], qk[..., hd // 2:]
    qk = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1).to(s["q"].dtype)
    s["q"].copy_(qk[:, :heads].reshape(s["rows"], heads * hd))
    slot = s["slot"].long()
    s["k_pool"][slot // page, :, slot % page] = qk[:, heads:]
    s["v_pool"][slot // page, :, slot % page] = x[:, heads + kv:].to(s["q"].dtype)


def _tokens(pool, table, count, most, page):
    """The first `most` tokens of every table as fp32 [tables][kv][most][hd], zero past a table's count, and which are there."""
    at = torch.arange(most, device="cuda")
    there = at < count.long()[:, None]
    page_of = torch.where(there, table.long()[:, at // page], 0)
    x = pool[page_of, :, at % page].float()                                # [tables][most][kv][hd]
    return torch.where(there[..., None, None], x, 0.0).transpose(1, 2), there


def _partial(q, k, v, seen):
    """Largest score, sum and weighted sum over the keys that `seen` leaves: q [..][kv][rows][hd], seen [..][1][rows][keys]."""
    score = torch.where(seen, q @ k.transpose(-1, -2), -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    return top, e.sum(-1, keepdim=True), e @ v


def _plain_attn(s):
    heads, kv, hd, page, n = s["heads"], s["kv"], s["hd"], s["page"], s["requests"]
    group, most, rows = heads // kv, s["most"], s["rows"]
    first, total = s["row_start"].long()[:-1], s["len"].long()
    new = s["row_start"].long()[1:] - first
    q = s["q"].float().view(rows, kv, group, hd) * hd ** -0.5

    def padded(start, count, width):
        """Rows start .. start + count of each item, as [items][kv][width * group][hd], and their numbers (rows: none)."""
        at = torch.arange(width, device="cuda")
        number = torch.where(at < count[:, None], start[:, None] + at, rows)
        x = q[number.clamp(max=rows - 1)]
        return x.permute(0, 2, 1, 3, 4).reshape(len(start), kv, width * group, hd), number

    def by_row(parts, number, width):
        """The parts of padded rows put back: [rows][kv][group][..]; rows that have none keep the empty sum."""
        out = []
        for x, empty in zip(parts, (-math.inf, 0.0, 0.0)):
            x = x.view(len(number), kv, width, group, -1).permute(0, 2, 1, 3, 4)
            y = torch.full((rows + 1,) + x.shape[2:], empty, device="cuda")
            y[number.reshape(-1)] = x.reshape((-1,) + x.shape[2:])
            out.append(y[:rows])
        return out

    k, _ = _tokens(s["k_pool"], s["table"], total, s["longest_own"], page)
    v, _ = _tokens(s["v_pool"], s["table"], total, s["longest_own"], page)
    x, number = padded(first, new, most)
    last = (total - new)[:, None] + torch.arange(most, device="cuda")
    seen = torch.arange(s["longest_own"], device="cuda") <= last[..., None]
    top, part, acc = by_row(_partial(x, k, v, seen.repeat_interleave(group, 1)[:, None]), number, most)
    if s["groups"]:
        k, there = _tokens(s["k_pool"], s["p_table"], s["prefix_len"], s["longest_prefix"], page)
        v, _ = _tokens(s["v_pool"], s["p_table"], s["prefix_len"], s["longest_prefix"], page)
        bounds = s["row_start"].long()[s["group_start"].long()]
        x, number = padded(bounds[:-1], bounds[1:] - bounds[:-1], s["most_group"])
        top2, part2, acc2 = by_row(_partial(x, k, v, there[:, None, None]), number, s["most_group"])
        both = torch.maximum(top, top2)
        a, b = torch.exp(top - both), torch.exp(top2 - both)
        part, acc = part * a + part2 * b, acc * a + acc2 * b
    s["out"].copy_((acc / part).view(rows, heads * hd))


# ------------------------------------------------------------------ the framework's calls

def _package():
    name = "llmb200"
    if name not in sys.modules:
        import importlib.util
        where = os.path.join(os.getcwd(), "llm.metal_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(where, "__init__.py"), submodule_search_locations=[where])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _arguments(s):
    """The filled argument structure of a call, which a program keeps beside its buffers, and the call."""
    pkg = _package()
    lib = pkg.lib()

    def fill(a, pointers, numbers):
        for field, tensor in pointers.items():
            setattr(a, field, tensor.data_ptr())
        for field, value in numbers.items():
            setattr(a, field, value)
        return a

    if s["op"] in ("extend", "release"):
        a = fill(pkg.PagesArgs(), dict(d_len=s["len"], d_len_out=s["len_out"], d_new=s["new"], d_base=s["base"], d_table=s["table"], d_free=s["free"], d_free_n=s["free_n"],
                                       d_free_n_out=s["free_n_out"], d_row_start=s["row_start"], d_slot=s["slot"], d_pos=s["pos"], d_status=s["status"]),
                 dict(n_req=s["requests"], page=s["page"], table_ld=s["table"].shape[1], n_pages=s["n_pages"], max_rows=s["slot"].numel()))
        return (lib.b200_pages_extend if s["op"] == "extend" else lib.b200_pages_release), a
    wtype = pkg.B200_WT_F16 if s["dtype"] == "f16" else pkg.B200_WT_BF16
    shape = dict(wtype=wtype, n_q=s["heads"], n_kv=s["kv"], hd=s["hd"], page=s["page"], n_pages=s["n_pages"], max_rows=s["rows"], q_ld=s["q"].shape[1])
    if s["op"] == "store":
        a = fill(pkg.PagedStoreArgs(), dict(d_qkv=s["qkv"], d_q_gamma=s["q_gamma"], d_k_gamma=s["k_gamma"], d_inv_freq=s["inv_freq"], d_rows=s["count"], d_slot=s["slot"],
                                            d_pos=s["pos"], d_k_pool=s["k_pool"], d_v_pool=s["v_pool"], d_q=s["q"]),
                 dict(eps=EPS, qkv_ld=s["qkv"].shape[1], **shape))
        return lib.b200_paged_store, a
    a = fill(pkg.PagedAttnArgs(), dict(d_q=s["q"], d_k_pool=s["k_pool"], d_v_pool=s["v_pool"], d_out=s["out"], d_row_start=s["row_start"], d_len=s["len"], d_table=s["table"],
                                       d_group_start=s["group_start"], d_prefix_len=s["prefix_len"], d_prefix_table=s["p_table"]),
             dict(scale=s["hd"] ** -0.5, out_ld=s["out"].shape[1], n_req=s["requests"], table_ld=s["table"].shape[1], n_groups=s["groups"], prefix_ld=s["p_table"].shape[1], **shape))
    size = lib.b200_paged_attn_work_bytes(C.byref(a))
    s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    a.d_work, a.work_bytes = s["work"].data_ptr(), size
    return lib.b200_paged_attn, a


def _call(s):
    if "call" not in s:
        s["call"] = _arguments(s)
    entry, a = s["call"]
    code = entry(C.byref(a), torch.cuda.current_stream().cuda_stream)
    if code:
        raise RuntimeError("%s: code %d" % (entry.__name__, code))


def run(s):
    if own:
        _call(s)
    else:
        {"extend": _plain_extend, "release": _plain_release, "store": _plain_store, "attn": _plain_attn}[s["op"]](s)
    if s["op"] == "extend":
        return {k: s[k] for k in ("table", "row_start", "slot", "pos", "len_out", "free_n_out")}
    if s["op"] == "release":
        return {k: s[k] for k in ("free", "free_n_out", "len_out")}
    if s["op"] == "store":
        return {k: s[k] for k in ("q", "k_pool", "v_pool")}
    return s["out"]


# ------------------------------------------------------------------ from the definition, in 64 bits

def _counted(s, page, extend):
    """The tables request by request, with a stack that is a list."""
    length, new, base, table = (s[k].tolist() for k in ("len", "new", "base", "table"))
    stack, left = s["free"].tolist(), s["free_n"].item()
    if not extend:
        free = stack[:left]
        for r, gone in enumerate(new):
            free += table[r][:_pages(length[r], page)] if gone else []
        return {"free": _ints(free + stack[len(free):]), "free_n_out": _ints([len(free)]), "len_out": _ints([0 if gone else t for t, gone in zip(length, new)])}
    free, rows, slot, pos = stack[:left], [0], [], []
    for r, more in enumerate(new):
        for token in range(length[r], length[r] + more):
            if token % page == 0:
                table[r][token // page] = free.pop()
            slot.append(table[r][token // page] * page + token % page)
            pos.append(base[r] + token)
        rows.append(len(slot))
    spare = [-1] * (s["slot"].numel() - len(slot))
    return {"table": _ints(table), "row_start": _ints(rows), "slot": _ints(slot + spare), "pos": _ints(pos + spare),
            "len_out": _ints([t + a for t, a in zip(length, new)]), "free_n_out": _ints([len(free)])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("extend", "release"):
        return _counted(s, case["page"], case["op"] == "extend")
    heads, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    if case["op"] == "store":
        x = s["qkv"].double().view(case["rows"], -1, hd)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None, None] * s["inv_freq"].double())

        def rotated(part, gamma):
            part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / hd + EPS) * gamma.double()
            z = torch.complex(part[..., :hd // 2], part[..., hd // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        pools = [torch.zeros(s["n_pages"] * page, kv, hd, dtype=torch.float64, device="cuda") for _ in range(2)]
        pools[0][s["slot"].long()] = rotated(x[:, heads:heads + kv], s["k_gamma"])
        pools[1][s["slot"].long()] = x[:, heads + kv:]
        k, v = (p.view(s["n_pages"], page, kv, hd).transpose(1, 2) for p in pools)
        return {"q": rotated(x[:, :heads], s["q_gamma"]).reshape(case["rows"], -1), "k_pool": k, "v_pool": v}
    total, new, starts, prefix = _lengths(case)
    if sum(total) + sum(p * (b - a) for p, a, b in zip(prefix, starts, starts[1:])) > 2 ** 23:
        return None                                                       # the keys of every request gathered on their own: minutes
    out, row = torch.zeros(s["rows"], heads, hd, dtype=torch.float64, device="cuda"), 0
    for r, (t, a) in enumerate(zip(total, new)):
        pages = [s["table"][r, :_pages(t, page)]]
        before = 0
        for g in range(len(prefix)):
            if starts[g] <= r < starts[g + 1] and prefix[g]:
                before = prefix[g]
                pages.insert(0, s["p_table"][g, :_pages(before, page)])
        cut = [before] * (len(pages) - 1) + [t]
        k, v = (torch.cat([pool[p.long()].transpose(0, 1).reshape(kv, -1, hd)[:, :c] for p, c in zip(pages, cut)], 1).double() for pool in (s["k_pool"], s["v_pool"]))
        x = s["q"][row:row + a].double().view(a, heads, hd)
        limit = before + t - a + torch.arange(a, device="cuda")
        for h in range(heads):
            z = (x[:, h] @ k[h * kv // heads].T) / math.sqrt(hd)
            z = z.masked_fill(torch.arange(before + t, device="cuda") > limit[:, None], -math.inf)
            out[row:row + a, h] = torch.softmax(z, -1) @ v[h * kv // heads]
        row += a
    return out.view(s["rows"], heads * hd)
