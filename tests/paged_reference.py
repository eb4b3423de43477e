"""Plain 64-bit forms of the paged operators, and caches to try them on.

Pages are shuffled, and what a row does not hold (the rest of its last page,
pages of nobody) is NaN, so that a read outside a row shows."""
import math
import random

import torch

PAGE, BLOCK, D = 256, 64, 128
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Cache:
    """Rows of given lengths in shuffled pages; ``spare`` pages more."""

    def __init__(self, lens, dtype, dev, seed=0, width=None, spare=3, fill=float("nan")):
        g = torch.Generator().manual_seed(seed)
        n_pages = [(n + PAGE - 1) // PAGE for n in lens]
        total = sum(n_pages) + spare
        ids = torch.randperm(total, generator=g).tolist()
        width = width or max(n_pages + [1]) + 1
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(n_pages):
            self.table[r, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        self.free = torch.tensor(ids[at:], dtype=torch.int32)
        kp = torch.full((total, PAGE, 1, D), fill)
        vp = torch.full((total, PAGE, 1, D), fill)
        self.k, self.v = [], []
        for r, n in enumerate(lens):
            k, v = torch.randn(n, D, generator=g).to(dtype), torch.randn(n, D, generator=g).to(dtype)
            for p in range(n_pages[r]):
                m = min(PAGE, n - p * PAGE)
                kp[self.table[r, p], :m, 0] = k[p * PAGE:p * PAGE + m].float()
                vp[self.table[r, p], :m, 0] = v[p * PAGE:p * PAGE + m].float()
            self.k.append(k)
            self.v.append(v)
        self.kp, self.vp = kp.to(dtype).to(dev), vp.to(dtype).to(dev)
        self.table, self.free = self.table.to(dev), self.free.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.free_ptr = torch.zeros(1, dtype=torch.int32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)

    def rows(self, r, n=None):
        """Keys and values of row r's first n tokens (default: all), from the pages, in 64 bits."""
        n = int(self.lens[r]) if n is None else n
        t = torch.arange(n, device=self.kp.device)
        page = self.table[r].long()[t // PAGE]
        return self.kp[page, t % PAGE, 0].double(), self.vp[page, t % PAGE, 0].double()


def softmax_rows(q, k, v, scale):
    """q [G, D], k, v [n, D] in 64 bits -> [G, D]; zeros without keys."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    return torch.softmax(q @ k.T * scale, -1) @ v


def attention_tolerance(dtype, q, ks, vs, scale, n):
    """Largest absolute error an output may have.

    A 16-bit type rounds the output and each probability (half a step each,
    relative); a logit is a 32-bit sum of 128 products (at most 128 half
    steps of 2^-24 of sum |q k|, twice in the exponent: in the row and in its
    maximum) and the exponential is 2^-22 off; a 32-bit sum of n terms of one
    sign is at most n half steps off, in numerator and denominator.  All of
    them scale with the largest |v|."""
    big = max([float(v.abs().max()) for v in vs if v.numel()] + [0.0])
    dot = max([float((q.abs() @ k.abs().T).max()) for q, k in zip(q, ks) if k.numel()] + [0.0])
    e = (130 * 2.0 ** -24 * dot * scale + 2.0 ** -22) * 2 + 2 * n * 2.0 ** -24
    if dtype != torch.float32:
        e += 2 * half_step(dtype)
    return e * big + 1e-30


def rotate(x, cos, sin):
    x = x.double()
    a, z = x[..., :64], x[..., 64:]
    c, s = cos.double(), sin.double()
    return torch.cat([a * c[..., :64] - z * s[..., :64], z * c[..., 64:] + a * s[..., 64:]], -1)


def block_scores(q, lo, hi):
    """q [G, D], lo, hi [blocks, D] -> the blocks' scores, in 64 bits."""
    q, lo, hi = q.double(), lo.double(), hi.double()
    s = torch.maximum(q[:, None] * lo, q[:, None] * hi).sum(-1)
    return torch.where(s.isnan(), math.inf, s).amax(0)


def pick(scores, n_select, sink, recent):
    m = len(scores)
    must = [j for j in range(m) if j < sink or j >= m - recent]
    rest = sorted((j for j in range(m) if j not in set(must)), key=lambda j: (-scores[j], j))
    return sorted((must + rest)[:n_select])


def rng_lens(n, lo, hi, seed):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]
