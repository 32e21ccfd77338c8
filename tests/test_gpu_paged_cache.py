"""Paged caches on the GPU: block tables and slots against lists, the cache's writer and the attention over pages against 64 bits, and a run of all of them."""
import ctypes as C
import math
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from _paged import TYPES, Step, args, ints  # noqa: E402


# ------------------------------------------------------------------ tables

class Tables:
    """A server's tables on the GPU beside the same ones as lists."""

    def __init__(self, pkg, n, page, table_ld, n_pages, max_rows, seed, base=True):
        self.lib, self.page, self.n_pages, self.max_rows = pkg.lib(), page, n_pages, max_rows
        rng = random.Random(seed)
        self.stack = list(range(n_pages))
        rng.shuffle(self.stack)
        self.lens, self.lists, self.bases = [0] * n, [[] for _ in range(n)], [rng.randrange(5000) for _ in range(n)]
        self.d = dict(len=ints([0] * n), new=ints([0] * n), base=ints(self.bases), table=torch.full((n, table_ld), -9, dtype=torch.int32, device="cuda"), free=ints(self.stack),
                      free_n=ints([n_pages]), row_start=torch.full((n + 1,), -9, dtype=torch.int32, device="cuda"), slot=torch.full((max_rows,), -9, dtype=torch.int32, device="cuda"),
                      pos=torch.full((max_rows,), -9, dtype=torch.int32, device="cuda"), status=ints([0]))
        d = self.d
        self.a = args(pkg.PagesArgs, n_req=n, page=page, table_ld=table_ld, n_pages=n_pages, max_rows=max_rows, d_len=d["len"], d_len_out=d["len"], d_new=d["new"],
                      d_table=d["table"], d_free=d["free"], d_free_n=d["free_n"], d_free_n_out=d["free_n"], d_row_start=d["row_start"], d_slot=d["slot"],
                      d_pos=d["pos"], d_status=d["status"], **(dict(d_base=d["base"]) if base else {}))
        if not base:
            self.bases = [0] * n

    def call(self, name, new):
        self.d["new"].copy_(ints(new))
        assert getattr(self.lib, name)(C.byref(self.a), None) == 0

    def extend(self, new):
        self.call("b200_pages_extend", new)
        rows, slot, pos = [0], [], []
        for r, more in enumerate(new):
            for token in range(self.lens[r], self.lens[r] + more):
                if token % self.page == 0:
                    self.lists[r].append(self.stack.pop())
                slot.append(self.lists[r][-1] * self.page + token % self.page)
                pos.append(self.bases[r] + token)
            self.lens[r] += more
            rows.append(len(slot))
        return rows, slot, pos

    def release(self, gone):
        self.call("b200_pages_release", gone)
        for r, g in enumerate(gone):
            if g:
                self.stack += self.lists[r]
                self.lists[r], self.lens[r] = [], 0

    def check(self, rows=None, slot=None, pos=None):
        d = {k: v.tolist() for k, v in self.d.items()}
        assert d["len"] == self.lens and d["free_n"] == [len(self.stack)] and d["free"][:len(self.stack)] == self.stack and d["status"] == [0]
        for r, mine in enumerate(self.lists):
            assert d["table"][r][:len(mine)] == mine
        if rows is not None:
            assert d["row_start"] == rows and d["slot"][:len(slot)] == slot and d["pos"][:len(pos)] == pos
            return d["slot"][len(slot):], d["pos"][len(pos):]


@pytest.mark.parametrize("n,page,most,max_rows", [(1, 16, 1, 1), (1, 256, 700, 700), (5, 16, 33, 165), (32, 16, 1, 32), (33, 64, 5, 200), (257, 32, 9, 2400), (1024, 16, 3, 2999), (1000, 16, 201, 150000)])
def test_extend_and_release_follow_the_lists(pkg, n, page, most, max_rows):
    rng = random.Random(n + page)
    t = Tables(pkg, n, page, 4 * (most // page + 2), n * 4 * (most // page + 2), max_rows, seed=n, base=n != 33)
    for step in range(4):
        new = [rng.choice([0, 1, most, rng.randint(0, most)]) for _ in range(n)]
        if step == 1:
            new = [0] * n
        rows, slot, pos = t.extend(new)
        spare_slot, spare_pos = t.check(rows, slot, pos)
        if step == 0:
            assert set(spare_slot + spare_pos) <= {-9}               # rows behind the last request's: as they were
        if step == 2:
            t.release([rng.choice([0, 0, 1, 5]) for _ in range(n)])
            t.check()
    t.release([1] * n)
    t.check()
    assert sorted(t.stack) == list(range(t.n_pages))


def test_extend_of_no_requests(pkg, lib):
    free_n, row_start = ints([3]), ints([-9])
    a = args(pkg.PagesArgs, n_req=0, page=16, table_ld=0, n_pages=3, max_rows=0, d_free=ints([0, 1, 2]), d_free_n=free_n, d_free_n_out=free_n, d_row_start=row_start)
    assert lib.b200_pages_extend(C.byref(a), None) == 0 and lib.b200_pages_release(C.byref(a), None) == 0
    assert free_n.tolist() == [3] and row_start.tolist() == [0]


@pytest.mark.parametrize("max_rows", [60, 5000])
@pytest.mark.parametrize("what,new,bits", [("pages", [40, 40, 40, 41], 1), ("table", [5, 97, 0, 1], 2), ("rows", [20, 20, 15, 6], 2), ("negative", [1, -1, 1, 1], 2), ("length", [1, 1, 1, 1], 2),
                                           ("length and height", [1, 1, 1, 1], 3), ("height", [1, 1, 1, 1], 1)])
def test_extend_is_all_or_nothing(pkg, max_rows, what, new, bits):
    if what == "rows" and max_rows > 60 or what == "pages" and max_rows == 60:
        pytest.skip("fits")
    t = Tables(pkg, 4, 16, 6, 10, max_rows, seed=1)
    t.extend([16, 1, 0, 7])
    if "length" in what:
        t.d["len"][2] = -3 if what == "length" else 97
    if "height" in what:
        t.d["free_n"][0] = 11 if what == "height" else -1
    before = {k: v.clone() for k, v in t.d.items()}
    t.call("b200_pages_extend", new)
    assert t.d["status"].tolist() == [bits] and t.d["row_start"].tolist() == [0] * 5
    for k in ("table", "slot", "pos", "len", "free", "free_n"):
        assert torch.equal(t.d[k], before[k]), k
    t.d["len"].copy_(ints(t.lens)); t.d["free_n"].copy_(ints([len(t.stack)])); t.d["status"].zero_()
    t.check(*t.extend([3, 3, 0, 1]))                                 # and goes on


def test_release_is_all_or_nothing(pkg):
    t = Tables(pkg, 3, 16, 6, 10, 64, seed=2)
    t.extend([40, 3, 3])
    t.d["free_n"][0] = 6                                             # 5 are out: 3 + 1 + 1 of 10
    before = {k: v.clone() for k, v in t.d.items()}
    t.call("b200_pages_release", [1, 1, 1])
    assert t.d["status"].tolist() == [1]
    assert all(torch.equal(t.d[k], before[k]) for k in ("table", "len", "free", "free_n"))
    t.d["free_n"][0] = 5; t.d["len"][1] = 6 * 16 + 1; t.d["status"].zero_()
    t.call("b200_pages_release", [0, 1, 0])
    assert t.d["status"].tolist() == [2] and t.d["free_n"].tolist() == [5]


def test_pages_outside_the_pool_give_no_slot(pkg):
    t = Tables(pkg, 2, 16, 6, 10, 64, seed=3)
    t.extend([5, 0])
    t.d["table"][0, 0] = 10                                          # the page that request 0 fills further
    t.d["free"][8] = -2                                              # the next one on the stack
    t.call("b200_pages_extend", [12, 3])
    assert t.d["status"].tolist() == [4]
    slot = t.d["slot"].tolist()
    assert slot[:12] == [-1] * 12 and all(0 <= s < 160 for s in slot[12:15])


@pytest.mark.parametrize("table_ld", [6, 600])                     # one block, and a cluster of them
@pytest.mark.parametrize("page_id", [-1, 10, 2 ** 31 - 1, -2 ** 31])
def test_release_reports_pages_outside_the_pool(pkg, page_id, table_ld):
    t = Tables(pkg, 4, 16, table_ld, 10, 64, seed=4)
    t.extend([5, 20, 3, 1])
    t.d["table"][0, 0] = page_id
    t.release([0, 1, 0, 1])                                          # not among them
    assert t.d["status"].tolist() == [0]
    t.lists[0][0] = page_id
    t.release([1, 0, 1, 0])
    assert t.d["status"].tolist() == [4]
    t.d["status"].zero_()
    t.check()                                                        # on the stack as it stood, and the rest in its place


# ------------------------------------------------------------------ the writer

def stored(pkg, dtype, n_q, n_kv, hd, page, rows, max_rows, pos, slots, n_pages, gamma=True, rotate=True, pad=0, seed=0):
    kind, wtype = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = (n_q + 2 * n_kv) * hd
    d = dict(qkv=torch.randn(max_rows, wide + 4 * pad, generator=g, device="cuda"), q=torch.full((max_rows, n_q * hd + 8 * pad), 7.0, dtype=kind, device="cuda"),
             k=torch.full((n_pages, n_kv, page, hd), 3.0, dtype=kind, device="cuda"), v=torch.full((n_pages, n_kv, page, hd), 5.0, dtype=kind, device="cuda"),
             qg=1 + 0.1 * torch.randn(hd, generator=g, device="cuda"), kg=1 + 0.1 * torch.randn(hd, generator=g, device="cuda"),
             freq=(1e6 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device="cuda") / hd)).float(), count=ints([rows]), pos=ints(pos), slot=ints(slots), status=ints([0]))
    a = args(pkg.PagedStoreArgs, wtype=wtype, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_pages=n_pages, max_rows=max_rows, eps=1e-6, d_qkv=d["qkv"], qkv_ld=d["qkv"].shape[1],
             d_rows=d["count"], d_slot=d["slot"], d_pos=d["pos"], d_k_pool=d["k"], d_v_pool=d["v"], d_q=d["q"], q_ld=d["q"].shape[1], d_status=d["status"],
             **(dict(d_q_gamma=d["qg"], d_k_gamma=d["kg"]) if gamma else {}), **(dict(d_inv_freq=d["freq"]) if rotate else {}))
    assert pkg.lib().b200_paged_store(C.byref(a), None) == 0

    def made(x, gam):
        x = x.double()
        if gamma:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gam.double()
        if rotate:
            t = d["pos"][:rows].double()[:, None, None] * d["freq"].double()
            lo, hi = x[..., :hd // 2], x[..., hd // 2:]
            x = torch.cat([lo * t.cos() - hi * t.sin(), lo * t.sin() + hi * t.cos()], -1)
        return x

    x = d["qkv"][:rows, :wide].view(rows, n_q + 2 * n_kv, hd)
    return d, made(x[:, :n_q], d["qg"]), made(x[:, n_q:n_q + n_kv], d["kg"]), x[:, n_q + n_kv:].double()


def near(got, want, pair):
    """One rounding to the type -- half a step, in binary16 at least 2^-25 -- of a sum of two products that are off by 2^-20 of the pair's length at most: norm (hd + 4
    roundings of a sum of squares, halved by the root: 2^-18 / 2 at hd 256 in the worst order; 2^-21 as shuffled), sine and cosine 2^-22, two products and a sum."""
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -19 * pair + tiny
    off = (got.double() - want).abs() / bound
    assert off.max() <= 1, off.max().item()


def length_of_pairs(x):
    half = x.shape[-1] // 2
    n = torch.sqrt(x[..., :half] ** 2 + x[..., half:] ** 2)
    return torch.cat([n, n], -1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,hd", [(8, 2, 64), (32, 8, 128), (4, 1, 256), (5, 5, 128), (1, 1, 64)])
@pytest.mark.parametrize("rows,max_rows,gamma,rotate,pad", [(1, 1, True, True, 0), (37, 40, True, True, 1), (37, 37, False, True, 0), (5, 600, True, False, 3), (530, 531, True, True, 0)])
def test_store(pkg, dtype, n_q, n_kv, hd, rows, max_rows, gamma, rotate, pad):
    page, n_pages = 16, 60
    rng = random.Random(rows)
    slots = rng.sample(range(page * n_pages), rows) + [0] * (max_rows - rows)
    pos = [rng.choice([0, 1, 17, 4095, 100003, 2 ** 24 + 1, 2 ** 29 - 1]) for _ in range(max_rows)]
    d, q, k, v = stored(pkg, dtype, n_q, n_kv, hd, page, rows, max_rows, pos, slots, n_pages, gamma, rotate, pad)
    near(d["q"][:rows, :n_q * hd].view(rows, n_q, hd), q, length_of_pairs(q))
    assert (d["q"][rows:] == 7).all() and (d["q"][:, n_q * hd:] == 7).all()
    at = d["slot"][:rows].long()
    near(d["k"][at // page, :, at % page], k, length_of_pairs(k))
    assert torch.equal(d["v"][at // page, :, at % page], v.to(d["v"].dtype))
    for pool, fill in ((d["k"], 3.0), (d["v"], 5.0)):
        pool[at // page, :, at % page] = fill
        assert (pool == fill).all()                                   # nothing else was written
    assert d["status"].tolist() == [0]


def test_store_leaves_out_slots_outside_the_pool(pkg):
    slots = [-1, 159, 160, 3, -2 ** 31, 2 ** 31 - 1]
    d, q, k, v = stored(pkg, "f16", 4, 2, 64, 16, 6, 6, [5] * 6, slots, 10)
    assert d["status"].tolist() == [4]
    near(d["q"].view(6, 4, 64), q, length_of_pairs(q))
    for row, s in ((1, 159), (3, 3)):
        assert torch.equal(d["v"][s // 16, :, s % 16], v[row].half())
        d["v"][s // 16, :, s % 16] = 5.0
    assert (d["v"] == 5).all()


@pytest.mark.parametrize("count", [-1, 7, 2 ** 31 - 1, -2 ** 31])
def test_store_of_a_count_that_does_not_fit(pkg, count):
    page, n_pages, max_rows = 16, 10, 6
    d, _, _, _ = stored(pkg, "f16", 4, 2, 64, page, max_rows, max_rows, [5] * 6, [1, 2, 3, 20, 50, 159], n_pages)
    for name, fill in (("q", 7.0), ("k", 3.0), ("v", 5.0)):
        d[name].fill_(fill)
    d["count"].fill_(count)
    a = args(pkg.PagedStoreArgs, wtype=1, n_q=4, n_kv=2, hd=64, page=page, n_pages=n_pages, max_rows=max_rows, eps=1e-6, d_qkv=d["qkv"], qkv_ld=d["qkv"].shape[1], d_rows=d["count"],
             d_slot=d["slot"], d_pos=d["pos"], d_k_pool=d["k"], d_v_pool=d["v"], d_q=d["q"], q_ld=d["q"].shape[1], d_status=d["status"])
    assert pkg.lib().b200_paged_store(C.byref(a), None) == 0
    assert d["status"].tolist() == [2]
    assert (d["q"] == 7).all() and (d["k"] == 3).all() and (d["v"] == 5).all()


@pytest.mark.parametrize("rows", [2, 40, 700])
def test_store_of_one_slot_for_all_rows(pkg, rows):
    """Every element is that of one of them, and nothing else is written."""
    page, n_pages = 16, 3
    d, _, k, v = stored(pkg, "bf16", 4, 2, 64, page, rows, rows, [9] * rows, [21] * rows, n_pages, rotate=False, gamma=False)
    for pool, fill, x in ((d["k"], 3.0, k), (d["v"], 5.0, v)):
        assert (pool[1, :, 5][None] == x.bfloat16()).any(0).all()
        pool[1, :, 5] = fill
        assert (pool == fill).all()


def test_store_behind_four_billion_elements(pkg):
    page, n_pages = 16, 2 ** 32 // (16 * 2 * 128) + 9                  # element offsets past 32 bits
    slots = [page * n_pages - 1, page * (n_pages - 8) + 3, 0]
    d, q, k, v = stored(pkg, "bf16", 2, 2, 128, page, 3, 3, [0, 1, 2], slots, n_pages)
    at = d["slot"].long()
    near(d["k"][at // page, :, at % page], k, length_of_pairs(k))
    assert torch.equal(d["v"][at // page, :, at % page], v.bfloat16())


# ------------------------------------------------------------------ attention

SHAPES = [(8, 2, 64), (32, 8, 128), (4, 1, 256), (5, 1, 128), (3, 3, 64), (64, 2, 64), (40, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,hd", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("total,new,groups,prefix", [
    ([1], [1], [], []),                                              # the first token of all
    ([17, 0, 1, 300, 64], [1, 0, 1, 1, 1], [], []),                  # a step without prefixes; a request that holds nothing
    ([1, 2, 33, 15], [1, 1, 1, 1], [0, 4], [513]),                   # one group
    ([5, 900, 16, 31, 7, 1], [1, 1, 1, 0, 1, 1], [1, 3, 3, 5], [129, 40, 0]),       # groups of unlike sizes, one empty, one without a prefix; requests outside them
    ([40, 3, 130], [7, 3, 129], [0, 2], [33]),                       # several new rows a request, causal
    ([8, 8, 8], [0, 0, 0], [0, 3], [50]),                            # nobody has a row
])
def test_attention(pkg, dtype, n_q, n_kv, hd, page, total, new, groups, prefix):
    s = Step(pkg, dtype, n_q, n_kv, hd, page, total, new, groups, prefix, seed=hd + page)
    s.run()
    s.check()
    assert s.status.tolist() == [0]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,hd,page,total,new,groups,prefix", [
    (32, 8, 128, 16, [700, 1, 90] * 11, [1] * 33, [0, 33], [4099]),              # a group of many rows: tiles that are full and one that is not
    (16, 2, 64, 32, [5, 250, 33, 1] * 25, [1, 2, 8, 1] * 25, [0, 1, 40, 100], [1000, 7, 2050]),
    (4, 1, 256, 128, [300, 200, 100], [290, 170, 5], [0, 3], [517]),             # portions
    (32, 8, 128, 64, [1000, 301], [640, 300], [0, 1], [1500]),
    (8, 8, 128, 256, [2000, 17], [129, 17], [0, 2], [128]),
    (5, 1, 128, 16, [260, 4000], [260, 77], [0, 2], [1]),
    (128, 1, 64, 16, [1, 2, 500], [1, 2, 3], [0, 3], [777]),                     # more query heads to a key / value head than a tile has rows
    (32, 8, 128, 16, [500, 700, 3, 90, 333], [1, 200, 1, 40, 31], [0, 4], [301]),         # portions and single tokens in one group
    (16, 2, 64, 32, [40, 64, 9, 1000, 17], [1, 64, 2, 16, 17], [1, 5], [640]),
    (8, 1, 128, 64, [16, 700, 16], [16, 500, 1], [0, 2, 3], [4000, 127]),
    (16, 8, 128, 16, [2] * 200 + [3000] * 24, [1] * 224, [0, 100, 224], [300, 90]),
])
def test_attention_larger(pkg, dtype, n_q, n_kv, hd, page, total, new, groups, prefix):
    s = Step(pkg, dtype, n_q, n_kv, hd, page, total, new, groups, prefix, seed=len(total))
    s.run()
    s.check()
    assert s.status.tolist() == [0]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_of_the_most_requests(pkg, dtype):
    rng = random.Random(5)
    new = [rng.choice([0, 1, 2]) for _ in range(1024)]
    total = [a + rng.randint(0, 60) for a in new]
    cuts = sorted(rng.sample(range(1, 1024), 510))
    s = Step(pkg, dtype, 4, 2, 64, 16, total, new, [0] + cuts + [1024], [rng.choice([0, 5, 100]) for _ in range(511)], seed=9)
    s.run()
    s.check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_the_most_groups(pkg, hd):
    """As many groups as requests: the largest plan, which leaves the fewest places for keys and values."""
    rng = random.Random(6)
    new = [rng.choice([0, 1, 1, 1, 9, 20]) if r % 50 else 70 for r in range(1024)]
    total = [a + rng.randint(0, 90) for a in new]
    s = Step(pkg, "f16", 4, 1, hd, 16, total, new, list(range(1025)), [rng.choice([0, 3, 200, 333]) for _ in range(1024)], seed=10)
    s.run()
    s.check()


@pytest.mark.parametrize("fill", [float("inf"), -float("inf"), 0.0])
def test_attention_with_other_unseen_slots(pkg, fill):
    s = Step(pkg, "f16", 8, 2, 128, 32, [33, 70, 5], [1, 40, 5], [0, 2], [100], fill=fill)
    s.run()
    s.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("n_q,n_kv,hd,new", [(8, 2, 128, 40), (8, 2, 64, 200), (4, 1, 256, 30), (2, 2, 128, 300)])
def test_values_that_only_later_rows_see(pkg, dtype, value, n_q, n_kv, hd, new):
    """Infinite values (and keys that are NaN) of new tokens: rows before them are as they would be without."""
    s = Step(pkg, dtype, n_q, n_kv, hd, 16, [new + 3], [new], [0, 1], [20])
    for token in (5, new // 2, new + 1):
        page, at = s.table[0, token // 16].long(), token % 16
        s.v[page, 0, at, 3:7] = value
        s.v[page, n_kv - 1, at, hd - 1] = -value
    s.k[s.table[0, (new + 2) // 16].long(), :, (new + 2) % 16, 0] = float("nan")
    s.run()
    s.check()


def test_scores_of_all_sizes(pkg):
    """Rows whose largest score comes last, first, or is far above all others; and zero queries, which weigh all keys alike."""
    for scale in (0.0, 30.0, -40.0):
        s = Step(pkg, "f16", 8, 2, 128, 16, [500, 260], [1, 130], [0, 2], [300], q_scale=scale)
        s.run()
        s.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd,new,n_req", [(64, 1, 148), (128, 1, 148), (256, 1, 74), (64, 40, 18), (128, 40, 18), (128, 200, 18)])
@pytest.mark.parametrize("shared", [False, True])
def test_one_strong_key_before_many_weak_ones(pkg, dtype, hd, new, n_req, shared):
    """8192 keys of 2^-26 of the first one's weight each make up all of the result, in tiles that few workers cut. Its error: the results' rounding and the weights' -- half a step of
    the type each, in binary16 at least half of its smallest number, 2^-25, where the largest weight is 2^15 (2^7 where there are many rows): 2^-40 (2^-32) of the largest each --,
    sums of n terms (n 2^-23), and the score, 18, by 2^-22 of it."""
    n, kv, value = 8192, 8, 8.0
    own = new if shared else n
    s = Step(pkg, dtype, kv, kv, hd, 128, [own] * n_req, [new] * n_req, range(n_req + 1) if shared else (), [n] * n_req if shared else (), scale=1.0)
    s.k.zero_(); s.v.fill_(value); s.q.zero_()
    strong, at = 16.0, (s.p_table if shared else s.table)[:, 0].long()
    s.k[at, :, 0, 0], s.v[at, :, 0] = strong, 0
    s.q.view(s.max_rows, kv, hd)[:, :, 0] = 26 * math.log(2) / strong
    s.run()
    assert s.status.tolist() == [0]
    score, eps = strong * s.q[0, 0].double().item(), torch.finfo(s.type).eps
    weak = (n if shared else n - new) + torch.arange(new, device="cuda").double()[:, None]     # keys that row i sees, without the strong one
    share = weak * math.exp(-score)
    want = value * share / (1 + share)
    tiny = (2.0 ** -40 if new == 1 else 2.0 ** -32) if dtype == "f16" else 0.0
    bound = want * (eps * 1.01 + 2 * score * 2.0 ** -22 + 2 * n * 2.0 ** -23) + tiny * weak * value
    off = (s.out[:s.rows].double().view(n_req, new, kv * hd) - want).abs() / bound
    assert off.max() <= 1, off.max().item()


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.7])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scales(pkg, scale, hd):
    s = Step(pkg, "bf16", 8, 2, hd, 128, [500, 260, 3], [1, 130, 3], [0, 3], [300], scale=scale)
    s.run()
    s.check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_of_all_sizes_hold_shared_prefixes(pkg, page, hd):
    for prefix in (1, 63, 64, 65, 257, 1000):
        s = Step(pkg, "f16", 16, 2, hd, page, [page, 1, page + 1, 2 * page - 1] * 3, [1] * 12, [0, 12], [prefix], seed=prefix)
        s.run()
        s.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,hd", [(16, 2, 64), (32, 8, 128), (4, 1, 256)])
@pytest.mark.parametrize("total,new", [([700, 90, 3], [1, 1, 1]), ([700, 0, 300], [1, 0, 140]), ([5, 5, 5], [0, 0, 0])])
def test_attention_of_few_rows_under_a_large_bound(pkg, dtype, n_q, n_kv, hd, total, new):
    s = Step(pkg, dtype, n_q, n_kv, hd, 16, total, new, [0, 3], [1000], max_rows=8192)
    s.run()
    s.check()
    assert s.status.tolist() == [0]


@pytest.mark.parametrize("q_pad,out_pad", [(8, 16), (136, 0)])
def test_attention_strides(pkg, q_pad, out_pad):
    s = Step(pkg, "bf16", 16, 8, 128, 16, [50, 300, 9], [1, 5, 9], [0, 3], [70], q_pad=q_pad, out_pad=out_pad, table_pad=5)
    s.run()
    s.check()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_behind_four_billion_elements(pkg, hd):
    first = 2 ** 32 // (64 * 2 * hd)
    s = Step(pkg, "bf16", 64, 2, hd, 64, [100, 3, 900], [1, 3, 200], [0, 2], [333], first_page=first, spare=0)
    s.run()
    s.check()
    assert s.k.numel() > 2 ** 32


def test_same_bits_again_and_on_another_stream(pkg):
    s = Step(pkg, "f16", 32, 8, 128, 16, [700, 130, 90, 2], [1, 100, 1, 1], [0, 4], [2000])
    want = s.run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        s.out.fill_(7.0); s.work.fill_(0xff)
        side.wait_stream(torch.cuda.current_stream())
        s.run(side.cuda_stream)
        side.synchronize()
        assert torch.equal(s.out, want)


def test_the_first_call_may_be_a_captured_one(pkg):
    """In a process of its own: nothing was launched before the capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys; sys.path[:0] = [%r, %r]\nimport torch, __graft_entry__ as e\nfrom _paged import Step\n"
            "s = Step(e.load_package(), 'f16', 8, 2, 128, 16, [40, 700], [1, 90], [0, 2], [100])\ntorch.cuda.synchronize()\ng = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g): s.run(torch.cuda.current_stream().cuda_stream)\n"
            "assert (s.out == 7).all()\nfor _ in range(3): g.replay()\ntorch.cuda.synchronize()\ns.check()\nprint('fine')\n") % (here, os.path.dirname(here))
    r = subprocess.run([sys.executable, "-c", code], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-2000:]


def test_two_calls_at_once(pkg):
    """On two streams, each with its own d_work: as alone."""
    steps = [Step(pkg, "bf16", 32, 8, 128, 16, [900, 1, 260] * 5, [1, 1, 60] * 5, [0, 15], [3000], seed=k) for k in (1, 2)]
    want = [s.run().clone() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for s in steps:
        s.out.fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, at in zip(steps, streams):
            s.run(at.cuda_stream)
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        assert torch.equal(s.out, w) and s.status.tolist() == [0]


@pytest.mark.parametrize("field,values", [
    ("d_row_start", [0, 3, 2, 4]), ("d_row_start", [1, 2, 3, 4]), ("d_row_start", [0, 1, 2, 60]), ("d_row_start", [0, -1, 2, 4]),
    ("d_len", [0, 5, 5]), ("d_len", [5, 5, -1]), ("d_len", [5, 16 * 3 + 1, 5]), ("d_group_start", [0, 4]), ("d_group_start", [2, 1]), ("d_group_start", [-1, 2]),
    ("d_prefix_len", [-1]), ("d_prefix_len", [16 * 4 + 1])])
def test_lengths_that_do_not_fit_change_nothing(pkg, field, values):
    s = Step(pkg, "f16", 8, 2, 64, 16, [20, 30, 32], [1, 2, 1], [0, 3], [40])
    assert s.a.table_ld == 3 and s.a.prefix_ld == 4 and s.max_rows == 6
    setattr(s.a, field, (kept := ints(values)).data_ptr())
    s.run()
    assert (s.out == 7).all() and s.status.tolist() == [2] and kept is not None


@pytest.mark.parametrize("page_id", [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("n_new", [1, 200])
def test_pages_outside_the_pool_are_not_read(pkg, page_id, n_new):
    """Rows that see none of them are right, and the status says so."""
    total, new = [220, 33, 300], [1, 1, n_new]
    s = Step(pkg, "f16", 32, 8, 128, 16, total, new, [0, 2], [70])
    s.table[2, 4] = page_id
    s.run()
    assert s.status.tolist() == [4]
    got = s.out.clone()
    s.new[2] = 0
    s.table[2, 4] = 0
    kept, s.rows = s.rows, s.ends[2]
    got[s.rows:kept] = 7.0
    s.check(got)


def test_one_capture_serves_growing_requests(pkg, lib):
    """A step as a program captures it -- tables, rows into their slots, attention -- and replays while requests grow, for two states at once: against attention over
    all that was ever stored, in 64 bits."""
    n_q, n_kv, hd, page, n, prefix = 8, 2, 128, 16, 3, 37
    states = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n_pages, p_pages = 64, 3
        d = dict(len=ints([0] * n), new=ints([1] * n), base=ints([prefix] * n), table=torch.full((n, 8), -1, dtype=torch.int32, device="cuda"), free=ints(range(p_pages, n_pages)),
                 free_n=ints([n_pages - p_pages]), row_start=ints([0] * (n + 1)), slot=ints([-1] * 30), pos=ints([-1] * 30), status=ints([0]),
                 qkv=torch.zeros(30, (n_q + 2 * n_kv) * hd, device="cuda"), q=torch.zeros(30, n_q * hd, dtype=torch.float16, device="cuda"), out=torch.zeros(30, n_q * hd, dtype=torch.float16, device="cuda"),
                 k=torch.zeros(n_pages, n_kv, page, hd, dtype=torch.float16, device="cuda"), v=torch.zeros(n_pages, n_kv, page, hd, dtype=torch.float16, device="cuda"),
                 freq=(1e4 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device="cuda") / hd)).float(), ptable=ints([0, 1, 2]), plen=ints([prefix]), group=ints([0, n]))
        d["k"][:p_pages].normal_(generator=g); d["v"][:p_pages].normal_(generator=g)
        pages = args(pkg.PagesArgs, n_req=n, page=page, table_ld=8, n_pages=n_pages, max_rows=30, d_len=d["len"], d_len_out=d["len"], d_new=d["new"], d_base=d["base"],
                     d_table=d["table"], d_free=d["free"], d_free_n=d["free_n"], d_free_n_out=d["free_n"], d_row_start=d["row_start"], d_slot=d["slot"], d_pos=d["pos"], d_status=d["status"])
        store = args(pkg.PagedStoreArgs, wtype=1, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_pages=n_pages, max_rows=30, eps=1e-6, d_qkv=d["qkv"], qkv_ld=d["qkv"].shape[1],
                     d_inv_freq=d["freq"], d_rows=d["row_start"][n:], d_slot=d["slot"], d_pos=d["pos"], d_k_pool=d["k"], d_v_pool=d["v"], d_q=d["q"], q_ld=n_q * hd, d_status=d["status"], use_pdl=1)
        attn = args(pkg.PagedAttnArgs, wtype=1, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_pages=n_pages, max_rows=30, scale=hd ** -0.5, d_q=d["q"], q_ld=n_q * hd, d_k_pool=d["k"], d_v_pool=d["v"],
                    d_out=d["out"], out_ld=n_q * hd, n_req=n, d_row_start=d["row_start"], d_len=d["len"], d_table=d["table"], table_ld=8, n_groups=1, d_group_start=d["group"],
                    d_prefix_len=d["plen"], d_prefix_table=d["ptable"], prefix_ld=3, d_status=d["status"], use_pdl=1)
        d["work"] = torch.empty(lib.b200_paged_attn_work_bytes(C.byref(attn)), dtype=torch.uint8, device="cuda")
        attn.d_work, attn.work_bytes = d["work"].data_ptr(), d["work"].numel()

        def step(pages=pages, store=store, attn=attn):
            at = torch.cuda.current_stream().cuda_stream
            assert lib.b200_pages_extend(C.byref(pages), at) == 0
            assert lib.b200_paged_store(C.byref(store), at) == 0
            assert lib.b200_paged_attn(C.byref(attn), at) == 0

        d["new"].zero_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()                                                    # without rows: nothing changes
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        states.append((d, graph, g, [[] for _ in range(n)], torch.cuda.Stream()))
    rng = random.Random(3)
    for turn in range(7):
        new = [[rng.choice([0, 1, 1, 10]) if turn else [4, 0, 10][r] for r in range(n)] for _ in states]
        for (d, graph, g, kept, stream), mine in zip(states, new):
            d["new"].copy_(ints(mine))
            d["qkv"].normal_(generator=g)
            stream.wait_stream(torch.cuda.current_stream())
        for _, graph, _, _, stream in states:                         # both graphs at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (d, graph, g, kept, stream), mine in zip(states, new):
            assert d["status"].tolist() == [0]
            row = 0
            for r, a in enumerate(mine):
                x = d["qkv"][row:row + a].double().view(a, n_q + 2 * n_kv, hd)
                length = sum(len(c[0]) for c in kept[r])
                angle = (prefix + length + torch.arange(a, device="cuda")).double()[:, None, None] * d["freq"].double()
                lo, hi = x[:, :n_q + n_kv, :hd // 2], x[:, :n_q + n_kv, hd // 2:]
                qk = torch.cat([lo * angle.cos() - hi * angle.sin(), lo * angle.sin() + hi * angle.cos()], -1)
                kept[r].append((qk[:, n_q:], x[:, n_q + n_kv:]))
                if a:
                    pk, pv = (p[:3].transpose(1, 2).reshape(48, n_kv, hd)[:prefix].double() for p in (d["k"], d["v"]))
                    k, v = (torch.cat([first] + [c[i] for c in kept[r]]) for i, first in ((0, pk), (1, pv)))
                    hidden = torch.arange(len(k), device="cuda") > (prefix + length + torch.arange(a, device="cuda"))[:, None]
                    for h in range(n_q):
                        z = (qk[:, h] @ k[:, h // 4].T * hd ** -0.5).masked_fill(hidden, -math.inf)
                        w = torch.softmax(z, -1)
                        # queries, keys and values are rounded to binary16 (2^-11 of each, so of a score at most 2^-10 of its terms' sum: e), weights and results too
                        e = 2.0 ** -10 * (qk[:, h].abs() @ k[:, h // 4].abs().T * hd ** -0.5).masked_fill(hidden, 0).amax(-1, keepdim=True) + 2.0 ** -18
                        bound = (2 * torch.expm1(e) + 3 * 2.0 ** -11) * (w @ v[:, h // 4].abs()) + 2.0 ** -14
                        got = d["out"][row:row + a, h * hd:(h + 1) * hd].double()
                        assert ((got - w @ v[:, h // 4]).abs() <= bound).all(), (turn, r, h)
                row += a
