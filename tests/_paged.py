"""What the tests of paged caches share: a step's buffers on the GPU, and its attention in 64 bits with the error that the kernels may have."""
import ctypes as C
import math

import torch

TYPES = {"f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def args(cls, **fields):
    """An argument structure; tensors stand for their addresses."""
    a = cls()
    for k, v in fields.items():
        setattr(a, k, v.data_ptr() if isinstance(v, torch.Tensor) else v)
    a._kept = fields                                          # the buffers live as long as the structure
    return a


class Step:
    """Pools, tables, rows and the argument structure of an attention call. `fill`: what unseen slots hold."""

    def __init__(self, pkg, dtype, n_q, n_kv, hd, page, total, new, groups=(), prefix=(), seed=0, fill=float("nan"), spare=3, q_scale=2.0,
                 first_page=0, q_pad=0, out_pad=0, table_pad=1, max_rows=None, scale=None):
        self.pkg, self.lib = pkg, pkg.lib()
        self.n_q, self.n_kv, self.hd, self.page, self.total, self.new = n_q, n_kv, hd, page, list(total), list(new)
        self.scale = hd ** -0.5 if scale is None else scale
        self.groups, self.prefix = list(groups), list(prefix)       # first request of every group and the end; prefixes
        self.type, wtype = TYPES[dtype]
        g = torch.Generator(device="cuda").manual_seed(seed)
        pages = lambda n: -(-n // page)                              # noqa: E731
        n_pages = first_page + sum(map(pages, self.total)) + sum(map(pages, self.prefix)) + spare
        order = (first_page + torch.randperm(n_pages - first_page, generator=g, device="cuda")).int()
        shape = (n_pages, n_kv, page, hd)
        self.k, self.v = (torch.full(shape, fill, dtype=self.type, device="cuda") if not first_page else torch.empty(shape, dtype=self.type, device="cuda") for _ in range(2))
        ld, p_ld = max(list(map(pages, self.total)) + [0]) + table_pad, max(list(map(pages, self.prefix)) + [0]) + table_pad
        at = 0

        def lay(counts, width):
            nonlocal at
            table = torch.full((max(1, len(counts)), width), -7, dtype=torch.int32, device="cuda")      # behind the last page: not read
            for i, n in enumerate(counts):
                ids = order[at:at + pages(n)]
                at += pages(n)
                table[i, :len(ids)] = ids
                for pool in (self.k, self.v):
                    x = torch.randn(n, n_kv, hd, generator=g, device="cuda").to(self.type)
                    where = torch.arange(n, device="cuda")
                    pool[ids.long()[where // page], :, where % page] = x
            return table

        self.table, self.p_table = lay(self.total, ld), lay(self.prefix, p_ld)
        self.ends = [0]
        for n in self.new:
            self.ends.append(self.ends[-1] + n)
        self.rows = self.ends[-1]
        self.max_rows = self.rows + 2 if max_rows is None else max_rows
        self.q = torch.full((self.max_rows, n_q * hd + q_pad), fill, dtype=self.type, device="cuda")
        self.q[:self.rows, :n_q * hd] = (q_scale * torch.randn(self.rows, n_q * hd, generator=g, device="cuda")).to(self.type)
        self.out = torch.full((self.max_rows, n_q * hd + out_pad), 7.0, dtype=self.type, device="cuda")
        self.status = ints([0])
        self.a = args(pkg.PagedAttnArgs, wtype=wtype, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_pages=n_pages, max_rows=self.max_rows, scale=self.scale,
                      d_q=self.q, q_ld=self.q.shape[1], d_k_pool=self.k, d_v_pool=self.v, d_out=self.out, out_ld=self.out.shape[1],
                      n_req=len(self.new), d_row_start=ints(self.ends), d_len=ints(self.total), d_table=self.table, table_ld=ld,
                      n_groups=len(self.prefix), d_group_start=ints(self.groups or [0]), d_prefix_len=ints(self.prefix or [0]), d_prefix_table=self.p_table, prefix_ld=p_ld,
                      d_status=self.status)
        self.own_work()

    def own_work(self):
        size = self.lib.b200_paged_attn_work_bytes(C.byref(self.a))
        assert size > 0
        self.work = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")          # NaN, whatever it is read as
        self.a.d_work, self.a.work_bytes = self.work.data_ptr(), size

    def run(self, stream=None):
        code = self.lib.b200_paged_attn(C.byref(self.a), stream)
        assert code == 0, code
        return self.out

    def keys(self, r):
        """Keys and values that request r's rows see, [kv][n][hd] in 64 bits, and how many of them are its group's."""
        parts, before = [], 0
        for g, p in enumerate(self.prefix):
            if self.groups[g] <= r < self.groups[g + 1] and p:
                parts, before = [(self.p_table[g], p)], p
        parts.append((self.table[r], self.total[r]))
        out = []
        for pool in (self.k, self.v):
            out.append(torch.cat([pool[t[:-(-n // self.page)].long()].transpose(0, 1).reshape(self.n_kv, -1, self.hd)[:, :n] for t, n in parts], 1).double())
        return out[0], out[1], before

    def check(self, got=None):
        """Against 64 bits. The error of a result, by arithmetic: weights are rounded to the type (half a step each, and in binary16 at least 2^-25 of the largest),
        the result once more; a score is a sum of hd products in fp32 (2^-23 of their magnitudes' sum an addition: the tensor cores truncate), times
        a constant rounded once, and so is off by at most e = (hd + 4) 2^-23 sum |q k| scale, a weight by a factor exp(2 e), with 2^-21 more for the exponential; sums of n
        terms in fp32 are off by n 2^-23 of their magnitudes."""
        got = self.out if got is None else got
        eps = torch.finfo(self.type).eps
        tiny = 2.0 ** -25 if self.type == torch.float16 else 0.0
        for r, a in enumerate(self.new):
            if not a:
                continue
            k, v, before = self.keys(r)
            q = self.q[self.ends[r]:self.ends[r + 1], :self.n_q * self.hd].double().view(a, self.n_q, self.hd)
            y = got[self.ends[r]:self.ends[r + 1], :self.n_q * self.hd].double().view(a, self.n_q, self.hd)
            hidden = torch.arange(k.shape[1], device="cuda") > (before + self.total[r] - a + torch.arange(a, device="cuda"))[:, None]
            kept_k, kept_v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
            for h in range(self.n_q):
                i = h // (self.n_q // self.n_kv)
                z = (q[:, h] @ k[i].T * self.scale).masked_fill(hidden, -math.inf)
                size = (q[:, h].abs() @ kept_k[i].abs().T * abs(self.scale)).masked_fill(hidden, 0)
                w = torch.softmax(z, -1)
                terms = torch.where(hidden[..., None], 0.0, w[..., None] * v[i]) if not torch.isfinite(v[i]).all() else None
                want = terms.sum(1) if terms is not None else w @ v[i]
                magnitude = w @ kept_v[i].abs()
                e = 2 * (self.hd + 4) * 2.0 ** -23 * size.amax(-1, keepdim=True) + 2.0 ** -21
                e = torch.expm1(e) * 2 + k.shape[1] * 2.0 ** -23
                total = torch.exp(z - z.amax(-1, keepdim=True)).sum(-1, keepdim=True)
                small = tiny * (~hidden).double() @ kept_v[i].abs() / total
                bound = (eps / 2 + e) * (1 + eps) * magnitude + small + eps / 2 * want.abs() + tiny
                fine = torch.isfinite(want)
                assert torch.equal(torch.isfinite(y[:, h]), fine), (r, h)
                off = ((y[:, h] - want).abs() / bound)[fine]
                assert off.numel() == 0 or off.max() <= 1, (r, h, off.max().item())
        assert (got[self.rows:] == 7.0).all()                        # rows behind the last request, and what lies between rows
        assert (got[:, self.n_q * self.hd:] == 7.0).all()
