"""The plan that attention over pages is cut by (csrc/paged_plan.cuh), laid on the host from the kernels' own source. The kernel that works on the keys and the one that joins
the pieces lay it each for itself, with 384 threads (128 above head dimension 128) and with 128: all of it has to come out the same, or pieces are looked for where none were left."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
FEW_MOST, BIG, BLOCKS = 32, 128, 148                          # as on a GPU of 148 SMs


@pytest.fixture(scope="module")
def laid(pkg, tmp_path_factory):
    """plan(threads, ...): the whole plan as a list, or None where the lengths are refused."""
    top = tmp_path_factory.mktemp("plan")
    at = top / "package" / "csrc"
    at.mkdir(parents=True)
    shutil.copytree(os.path.join(ROOT, "include"), top / "include")
    for f in ("host_block.h", "plan_on_host.cpp"):
        shutil.copy(os.path.join(HERE, f), at)
    shutil.copy(os.path.join(ROOT, "llm.metal_b200", "csrc", "paged_plan.cuh"), at / "paged_plan.cuh")
    (at / "stream_core.cuh").write_text("#pragma once\n")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wno-unknown-pragmas", "-shared", "-fPIC", str(at / "plan_on_host.cpp"), "-o", str(at / "plan.so")], check=True)
    lib = C.CDLL(str(at / "plan.so"))

    def plan(threads, new, total, starts=(), prefix=(), n_q=8, n_kv=1, page=16, ratio=16, few_warps=8, few_most=FEW_MOST, big=BIG):
        n, m = len(new), len(prefix)
        ints = lambda x: (C.c_int * max(1, len(x)))(*x)           # noqa: E731
        rows = [0]
        for x in new:
            rows.append(rows[-1] + x)
        kept = [ints(rows), ints(total), ints(list(starts) or [0]), ints(list(prefix) or [0])]
        status = C.c_uint(0)
        a = pkg.PagedAttnArgs(n_q=n_q, n_kv=n_kv, page=page, max_rows=max(1, rows[-1]), n_req=n, n_groups=m, table_ld=1 << 20, prefix_ld=1 << 20)
        for field, x in zip(("d_row_start", "d_len", "d_group_start", "d_prefix_len"), kept):
            setattr(a, field, C.addressof(x))
        a.d_status = C.addressof(status)
        out = (C.c_int * (5 + 4 * (n + m + 1) + n + 1))()
        fine = lib.plan_on_host(C.byref(a), few_most, big, BLOCKS, few_warps, ratio, threads, out)
        assert status.value == (0 if fine else pkg.B200_PAGED_BAD_LENGTH)
        return list(out) if fine else None

    return plan


def step(rng, n, groups, most):
    new = [rng.randint(0, most) for _ in range(n)]
    total = [a + rng.randint(0, 3000) for a in new]
    starts = sorted(rng.sample(range(n + 1), groups + 1)) if groups else []
    return dict(new=new, total=total, starts=starts, prefix=[rng.choice([0, 100, rng.randint(1, 9000)]) for _ in range(groups)])


@pytest.mark.parametrize("n,groups,most", [(1, 0, 1), (3, 2, 200), (40, 5, 8), (129, 0, 8), (200, 60, 8), (500, 3, 20), (1024, 1024 // 2, 8), (1024, 1023, 3)])
def test_both_kernels_lay_the_same_plan(laid, n, groups, most):
    rng = random.Random(n + groups)
    for _ in range(12):
        s = step(rng, n, groups, most)
        heads = rng.choice([(8, 1), (16, 2), (32, 8), (5, 5)])
        assert laid(384, **s, n_q=heads[0], n_kv=heads[1]) == laid(128, **s, n_q=heads[0], n_kv=heads[1])


@pytest.mark.parametrize("n,seed", [(600, 2), (1000, 3), (1000, 4)])
def test_both_kernels_divide_the_blocks_alike(laid, n, seed):
    """Where the second way's share of the work lies next to the border between two numbers of blocks: the work of one request more of the first way is moved over the border in the
    smallest steps."""
    rng = random.Random(seed)
    new = [rng.randint(5, 8) for _ in range(n)]                   # 40 .. 64 query rows: a tile of one stream each
    total = [rng.randint(10 ** 6, 2 * 10 ** 6) for _ in range(n)]

    def both(first):
        plans = [laid(t, [1] + new, [first] + total, page=256) for t in (384, 128)]
        assert plans[0] == plans[1], first
        return plans[0][0]

    lo, hi = 16, 1 << 28                                          # tokens of that request
    most = both(lo)
    for want in range(most, most - 4, -1):                        # the last length that still leaves the second way `want` blocks
        a, b = lo, hi
        if both(b) >= want:
            continue
        while b - a > 16:
            mid = (a + b) // 2
            a, b = (mid, b) if both(mid) >= want else (a, mid)
        for first in range(a - 40 * 16, a + 40 * 16, 16):
            if first > 0:
                both(first)


@pytest.mark.parametrize("rows,n_q,n_kv,wide,fits", [(131072, 32, 8, False, True), (180000, 32, 8, False, True), (190000, 32, 8, False, False), (1 << 20, 8, 1, True, True),
                                                     (1 << 20, 56, 8, True, True), (1 << 20, 128, 8, True, False), (1 << 20, 1024, 1, True, False), (1 << 20, 1024, 1024, False, False)])
def test_lines_are_refused_from_two_to_the_31_units_on(laid, rows, n_q, n_kv, wide, fits):
    """A prompt as one portion: tiles of 256 rows by units of 64 keys, or, above head dimension 128, of 16 by 16, of which a row's tile sees half on average."""
    tile, unit, gap = (256, 64, 8) if wide else (16, 16, 2)
    tiles = -(-rows * (n_q // n_kv) // tile)
    units = n_kv * sum(gap + 1 + (min((t + 1) * tile // (n_q // n_kv), rows)) / unit for t in range(0, tiles, 64)) * 64      # (every 64th tile stands for its neighbours)
    assert abs(units / 2 ** 31 - 1) > 0.01 and (units < 2 ** 31) == fits
    for threads in (384, 128):
        plan = laid(threads, [rows], [rows], n_q=n_q, n_kv=n_kv, **({} if wide else dict(few_most=2 ** 31 - 1, big=2 ** 31 - 1, few_warps=4)))
        assert (plan is not None) == fits
        if fits:
            assert abs(plan[4 if wide else 3] / units - 1) < 0.01
