"""A paged cache of 8 bits for tests: the quantising plainly in 64 bits, and pages with what a long-running server leaves in them."""
import torch

_E4M3 = torch.tensor([m / 512 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)], dtype=torch.float64)
LEAST, MOST = -15, 7


def times_power(x, e):
    """x 2^e in 64 bits, e from -15 to 15. (By a table: powers that a GPU computes need not be exact.)"""
    return x.double() * torch.tensor([2.0 ** i for i in range(-15, 16)], dtype=torch.float64, device=x.device)[e + 15]


def quantised(x):
    """(numbers of e4m3 in 64 bits, exponents) of rows [..., D]."""
    x = x.double()
    finite = x.isfinite()
    size = torch.where(finite, x.abs(), 0.0)
    holds = torch.tensor([448 * 2.0 ** i for i in range(LEAST, MOST)], dtype=torch.float64, device=x.device)
    e = LEAST + (size.amax(-1, keepdim=True) > holds).sum(-1)
    size = times_power(size, -e[..., None]).clamp(max=448).contiguous()
    table = _E4M3.to(x.device)
    above = torch.searchsorted(table, size).clamp(1, len(table) - 1)
    low, high = size - table[above - 1], table[above] - size
    up = (high < low) | ((high == low) & (above % 2 == 0))
    q = torch.copysign(table[torch.where(up, above, above - 1)], x)
    return torch.where(finite, q, torch.nan), e


class Cache8:
    """Every slot that holds no token of a sequence has NaN and a scale that is none."""

    def __init__(self, lens, Hk, D, page, dtype, seed, order="phd", spare=3, std=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page = lens, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
        self.table[:, -1] = 1 << 30
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(perm[at: at + n])
            at += n
        self.table = self.table.cuda()
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        # rows of very different sizes: a scale each
        size = torch.ldexp(torch.full((sum(lens), Hk, 1), std, device="cuda"), torch.randint(-3, 2, (sum(lens), Hk, 1), generator=gen, device="cuda"))
        self.k_rows, self.v_rows = ((torch.randn(sum(lens), Hk, D, generator=gen, device="cuda") * size).to(dtype) for _ in range(2))
        self.first = [sum(lens[:b]) for b in range(len(lens))]
        shape = {"phd": (pages, page, Hk, D), "hpd": (pages, Hk, page, D)}[order]
        self.k_pages, self.v_pages = (torch.full(shape, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
        if order == "hpd":
            self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        self.k_scales, self.v_scales = (torch.full((pages, Hk, page), 255, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2))
        (k, ke), (v, ve) = quantised(self.k_rows), quantised(self.v_rows)
        self.k, self.v = times_power(k, ke[..., None]), times_power(v, ve[..., None])  # what the cache stands for
        self.parts = k, ke, v, ve

    def args(self):
        return self.k_pages, self.v_pages, self.table, self.kv_lens

    def scales(self):
        return dict(k_scales=self.k_scales, v_scales=self.v_scales)

    def places(self, b, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        return self.table[b].long()[at // self.page], at % self.page

    def fill(self):
        k, ke, v, ve = self.parts
        for b, n in enumerate(self.lens):
            (page, slot), rows = self.places(b, 0, n), slice(self.first[b], self.first[b] + n)
            for pages, scales, x, e in ((self.k_pages, self.k_scales, k, ke), (self.v_pages, self.v_scales, v, ve)):
                pages.view(torch.uint8)[page, slot] = x[rows].float().to(torch.float8_e4m3fn).view(torch.uint8)
                scales.view(torch.uint8)[page, :, slot] = (e[rows] + 127).to(torch.uint8)
        return self
