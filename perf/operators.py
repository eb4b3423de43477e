"""What is measured of the paged cache's operators, and their plain forms.

Three operators over a cache of 256-token pages, [n_pages, 256, 1, 128] for keys and for values, with a page table
and a length for each row (sequence, KV head):

* ``append``: ``ops.rope_append`` rotates the new queries and keys, and puts the keys and values in their pages;
* ``shared``: ``ops.flash_decode_shared``, one query token a sequence, over a prefix that all sequences share (its
  pages are read once) and each sequence's own tail;
* ``sparse``: ``ops.flash_decode_sparse``, one query token a sequence, over the 64-token blocks that a bound on
  their scores selects.

Lengths and page tables follow from the case alone, values from the seed.
"""
import math
import random

import torch

own = False

PAGE, BLOCK, D = 256, 64, 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decode step of one sequence of an 8B model: latency
        dict(name="append-1x1", op="append", dtype="bf16", bsz=1, heads=32, kv=8, tokens=1, past=700, ragged=False,
             bounds=False),
        # one decode step of a serving batch, block bounds kept up to date
        dict(name="append-64x1", op="append", dtype="bf16", bsz=64, heads=32, kv=8, tokens=1, past=2000,
             ragged=False, bounds=True),
        # drafted tokens of a batch, not the same number for every sequence
        dict(name="append-17x5", op="append", dtype="fp16", bsz=17, heads=28, kv=4, tokens=5, past=1500, ragged=True,
             bounds=True),
        # a chunk of a long prompt for a batch
        dict(name="append-16x4096", op="append", dtype="bf16", bsz=16, heads=32, kv=8, tokens=4096, past=5000,
             ragged=True, bounds=True),
        # a few samples of a short prompt: latency
        dict(name="shared-3x1000", op="shared", dtype="bf16", bsz=3, heads=32, kv=8, prefix=1000, tail=70),
        # sixteen samples of a long prompt
        dict(name="shared-16x32k", op="shared", dtype="bf16", bsz=16, heads=32, kv=8, prefix=32768, tail=500),
        # a large batch of continuations at the longest prompt
        dict(name="shared-64x128k", op="shared", dtype="bf16", bsz=64, heads=32, kv=8, prefix=131072, tail=1000),
        # seven query heads a KV head, odd sizes
        dict(name="shared-29x20001", op="shared", dtype="fp16", bsz=29, heads=28, kv=4, prefix=20001, tail=333),
        # a 32-bit model
        dict(name="shared-6x3000", op="shared", dtype="fp32", bsz=6, heads=32, kv=8, prefix=3000, tail=100),
        # one sequence at the longest prompt
        dict(name="sparse-1x128k", op="sparse", dtype="bf16", bsz=1, heads=32, kv=8, length=131072, select=64, sink=1,
             recent=2),
        # a serving batch of long sequences
        dict(name="sparse-16x64k", op="sparse", dtype="bf16", bsz=16, heads=32, kv=8, length=65536, select=64, sink=1,
             recent=2),
        # seven query heads a KV head, odd sizes
        dict(name="sparse-5x9001", op="sparse", dtype="fp16", bsz=5, heads=28, kv=4, length=9001, select=33, sink=0,
             recent=1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "shared", "sparse"])
    heads, kv = rng.choice([(32, 8), (28, 4), (8, 8), (64, 8)])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), heads=heads, kv=kv)
    if op == "append":
        bsz = _log(rng, 1, 64)
        tokens = rng.choice([1, _log(rng, 1, min(8192, 60000 // bsz))])
        c.update(bsz=bsz, tokens=tokens, past=_log(rng, 1, 5000), ragged=rng.random() < 0.5,
                 bounds=rng.random() < 0.7)
    elif op == "shared":
        bsz = _log(rng, 1, 64)
        c.update(bsz=bsz, prefix=_log(rng, 1, min(131072, 260000000 // bsz // heads)), tail=_log(rng, 1, 1000))
    else:
        bsz = _log(rng, 1, 16)
        select = _log(rng, 4, 96)
        c.update(bsz=bsz, length=_log(rng, 60, min(131072, 1000000 // bsz)), select=select, sink=rng.randint(0, 2),
                 recent=rng.randint(1, 2))
    return c


# ---- what a case's lengths are

def _lengths(case):
    """Row lengths of the cache before the call, and the counts (append) or shared lengths (shared)."""
    r = random.Random("%(op)s-%(dtype)s-%(bsz)d-%(heads)d-%(kv)d" % case)
    b, kv = case["bsz"], case["kv"]
    if case["op"] == "append":
        past = [r.randint(case["past"] // 2, case["past"]) for _ in range(b * kv)]
        count = [r.randint((case["tokens"] + 1) // 2, case["tokens"]) if case["ragged"] else case["tokens"]
                 for _ in range(b)]
        return past, count
    if case["op"] == "shared":
        # some heads are kept whole, the others compressed
        shared = [max(1, int(case["prefix"] * (1.0 if h % 2 else r.uniform(0.2, 0.6)))) for h in range(kv)]
        return [shared[h] + r.randint(case["tail"] // 2, case["tail"]) for _ in range(b) for h in range(kv)], shared
    return [max(1, int(case["length"] * r.uniform(0.6, 1.0))) for _ in range(b * kv)], None


def _cuda(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 13)
    dt = DTYPES[case["dtype"]]
    b, heads, kv = case["bsz"], case["heads"], case["kv"]
    lens, extra = _lengths(case)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=dt)  # noqa: E731
    pages_of = lambda n: (n + PAGE - 1) // PAGE  # noqa: E731
    s = dict(case=case, dtype=dt, err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    r = random.Random(int(seed))
    if case["op"] == "append":
        T = case["tokens"]
        ends = [n + extra[i // kv] for i, n in enumerate(lens)]
        total = sum(pages_of(n) for n in ends)
        width = max(pages_of(n) for n in ends) + 1
        mapped = [pages_of(n) for n in lens]
    elif case["op"] == "shared":
        width = max(pages_of(n) for n in lens)
        total = sum(pages_of(n) for n in extra) + sum(pages_of(n) - extra[i % kv] // PAGE for i, n in enumerate(lens))
        mapped = None
    else:
        width = max(pages_of(n) for n in lens)
        total = sum(pages_of(n) for n in lens)
        mapped = [pages_of(n) for n in lens]
    total += 3
    ids = list(range(total))
    r.shuffle(ids)
    # neighbouring tokens' keys are alike: each block of 64 has a direction of its own
    kp = rnd(total, PAGE, 1, D)
    kp.view(total, PAGE // BLOCK, BLOCK, D).add_(rnd(total, PAGE // BLOCK, 1, D))
    s.update(kp=kp, vp=rnd(total, PAGE, 1, D))
    table = torch.full((b * kv, width), -1, dtype=torch.int32)
    at = 0
    if mapped is not None:
        for i, n in enumerate(mapped):
            table[i, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
    else:
        # a shared page is every sequence's; the page in which the prefix ends is copied for each
        for h in range(kv):
            n = pages_of(extra[h])
            table[h::kv, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        for i, n in enumerate(lens):
            first = extra[i % kv] // PAGE
            n = pages_of(n) - first
            if i < kv and extra[i] % PAGE:  # the first sequence keeps that page
                table[i, first + 1:first + n] = torch.tensor(ids[at:at + n - 1], dtype=torch.int32)
                at += n - 1
                continue
            table[i, first:first + n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
    s.update(table=table.cuda(), lens=_cuda(lens))
    if case["op"] == "append":
        # as the projections leave them: [bsz, tokens, heads, D] seen as [bsz, heads, tokens, D]
        s.update(q=rnd(b, T, heads, D).transpose(1, 2), k=rnd(b, T, kv, D).transpose(1, 2),
                 v=rnd(b, T, kv, D).transpose(1, 2))
        pos = torch.arange(T, device="cuda", dtype=torch.float64)[None] + 1000.0 * _cuda(
            [r.randint(0, 100) for _ in range(b)], torch.float64)[:, None]
        angle = pos[..., None] * 500000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        angle = torch.cat([angle, angle], -1)
        s.update(cos=angle.cos().to(dt), sin=angle.sin().to(dt), q_out=torch.zeros(b, heads, T, D, dtype=dt, device="cuda"),
                 free=torch.tensor(ids[at:], dtype=torch.int32).cuda(), free_ptr=_cuda([0]),
                 lens_out=torch.zeros(b * kv, dtype=torch.int32, device="cuda"),
                 counts=_cuda(extra) if case["ragged"] else None, bounds=None)
        if case["bounds"]:
            s["bounds"] = torch.zeros(total, PAGE // BLOCK, 2, D, dtype=dt, device="cuda")
            _plain_bounds(s["kp"], s["table"], s["lens"], s["bounds"])
    else:
        s.update(q=rnd(b, heads, 1, D))
        if case["op"] == "shared":
            s["shared"] = _cuda(extra)
        else:
            s["bounds"] = torch.zeros(total, PAGE // BLOCK, 2, D, dtype=dt, device="cuda")
            _plain_bounds(s["kp"], s["table"], s["lens"], s["bounds"])
    return s


# ---- the calls

def run(s):
    return {"append": run_append, "shared": run_shared, "sparse": run_sparse}[s["case"]["op"]](s)


def _workspace(s):
    if "workspace" not in s:
        from heterocache_b200.ops import Workspace
        s["workspace"] = Workspace(s["err"].device)
    return s["workspace"]


def run_append(s):
    if own:
        from heterocache_b200 import ops
        ops.rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["kp"], s["vp"], s["table"], s["lens"], s["free"],
                        s["free_ptr"], s["err"], workspace=_workspace(s), counts=s["counts"], q_out=s["q_out"],
                        heads_len_out=s["lens_out"], bounds=s["bounds"])
    else:
        plain_append(s)
    out = {n: s[n] for n in ("q_out", "kp", "vp", "table", "lens_out", "free_ptr")}
    if s["bounds"] is not None:
        out["bounds"] = s["bounds"]
    return out


def run_shared(s):
    if own:
        from heterocache_b200 import ops
        return ops.flash_decode_shared(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["shared"],
                                       num_kv_heads=s["case"]["kv"], workspace=_workspace(s), err=s["err"])
    return plain_shared(s)


def run_sparse(s):
    c = s["case"]
    if own:
        from heterocache_b200 import ops
        out, blocks, counts = ops.flash_decode_sparse(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["bounds"],
                                                      num_kv_heads=c["kv"], n_select=c["select"], sink=c["sink"],
                                                      recent=c["recent"], workspace=_workspace(s), err=s["err"])
        return {"out": out, "blocks": blocks, "counts": counts}
    return plain_sparse(s)


# ---- plain forms

def _rotate(x, cos, sin):
    x = x.float()
    half = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    return x * cos.float()[:, None] + half * sin.float()[:, None]


def _plain_bounds(kp, table, lens, bounds, first=None):
    """Least and greatest key of each block of a row's tokens, from the block of token ``first`` on."""
    width = table.shape[1] * (PAGE // BLOCK)
    j = torch.arange(width, device=lens.device)[None]
    lo = torch.zeros_like(lens) if first is None else first // BLOCK
    want = (j >= lo[:, None]) & (j * BLOCK < lens[:, None])
    row, blk = want.nonzero(as_tuple=True)
    page, part = table[row, blk // (PAGE // BLOCK)].long(), blk % (PAGE // BLOCK)
    keys = kp.view(-1, PAGE // BLOCK, BLOCK, D)[page, part]
    there = (blk[:, None] * BLOCK + torch.arange(BLOCK, device=lens.device)[None] < lens[row][:, None])[..., None]
    bounds[page, part, 0] = torch.where(there, keys, math.inf).amin(1)
    bounds[page, part, 1] = torch.where(there, keys, -math.inf).amax(1)


def plain_append(s):
    b, heads, T, _ = s["q"].shape
    kv = s["k"].shape[1]
    counts = s["counts"] if s["counts"] is not None else torch.full((b,), T, dtype=torch.int32, device="cuda")
    t = torch.arange(T, device="cuda")
    there = t[None] < counts[:, None]
    s["q_out"].copy_(torch.where(there[:, None, :, None], _rotate(s["q"], s["cos"], s["sin"]).to(s["dtype"]), s["q_out"]))
    n = counts.repeat_interleave(kv)
    end = s["lens"] + n
    # pages: the unmapped ones that a row reaches, in the order of the table
    col = torch.arange(s["table"].shape[1], device="cuda")[None]
    need = (col >= (s["lens"] // PAGE)[:, None]) & (col * PAGE < end[:, None]) & (s["table"] < 0)
    order = need.flatten().cumsum(0).view(need.shape) - 1 + s["free_ptr"].long()
    s["table"].copy_(torch.where(need, s["free"][order.clamp(0, s["free"].numel() - 1)], s["table"]))
    s["free_ptr"] += need.sum().int()
    row, tok = (there.repeat_interleave(kv, 0)).nonzero(as_tuple=True)
    pos = s["lens"][row].long() + tok
    page, slot = s["table"][row, pos // PAGE].long(), pos % PAGE
    k = _rotate(s["k"], s["cos"], s["sin"]).to(s["dtype"])
    s["kp"][page, slot, 0] = k[row // kv, row % kv, tok]
    s["vp"][page, slot, 0] = s["v"][row // kv, row % kv, tok]
    s["lens_out"].copy_(end)
    if s["bounds"] is not None:
        _plain_bounds(s["kp"], s["table"], end, s["bounds"], s["lens"])


def _attend(scores, there):
    """exp(scores - max) over the last axis where ``there``, and its sum; rows with nothing are zero."""
    scores = torch.where(there, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-37)


def plain_shared(s):
    b, heads, _, _ = s["q"].shape
    kv = s["case"]["kv"]
    G = heads // kv
    q = s["q"].float().view(b, kv, G, D).transpose(0, 1)  # [kv, b, G, D]
    width = int(s["table"].shape[1])
    tail = s["case"]["tail"]
    pages = (s["case"]["prefix"] + PAGE - 1) // PAGE
    first = s["table"][:kv, :pages].long().clamp_min(0)
    k = s["kp"][first].float().view(kv, pages * PAGE, D)
    v = s["vp"][first].float().view(kv, pages * PAGE, D)
    at = torch.arange(pages * PAGE, device="cuda")
    front = (at[None] < s["shared"][:, None])[:, None, None]
    a = torch.matmul(q.reshape(kv, b * G, D), k.transpose(1, 2)).view(kv, b, G, -1) / math.sqrt(D)
    # each row's own tokens, behind the shared ones
    pos = s["shared"].repeat(b)[:, None].long() + torch.arange(tail, device="cuda")[None]  # [rows, tail]
    back = (pos < s["lens"][:, None]).view(b, kv, 1, tail).transpose(0, 1)
    page = s["table"].gather(1, (pos // PAGE).clamp_max(width - 1)).long().clamp_min(0)
    kt = s["kp"][page, pos % PAGE, 0].float().view(b, kv, tail, D).transpose(0, 1)
    vt = s["vp"][page, pos % PAGE, 0].float().view(b, kv, tail, D).transpose(0, 1)
    c = torch.matmul(q, kt.transpose(2, 3)) / math.sqrt(D)
    p = _attend(torch.cat([a, c], -1), torch.cat([front.expand_as(a), back.expand_as(c)], -1))
    out = torch.matmul(p[..., :pages * PAGE].reshape(kv, b * G, -1), v).view(kv, b, G, D) + torch.matmul(
        p[..., pages * PAGE:], vt)
    return out.transpose(0, 1).reshape(b, heads, D).to(s["dtype"])


def plain_sparse(s):
    c = s["case"]
    b, heads, _, _ = s["q"].shape
    kv, n = c["kv"], c["select"]
    G, rows = heads // kv, b * kv
    per = PAGE // BLOCK
    pages = s["table"].long().clamp_min(0)
    width = pages.shape[1] * per
    bound = s["bounds"][pages].view(rows, width, 2, D).double()
    q = s["q"].double().view(rows, G, D)
    # sum of max(q lo, q hi): the sign of q says which; 64 bits, since which block is in must not hang on rounding
    score = torch.matmul(q.clamp_min(0), bound[:, :, 1].transpose(1, 2)) + torch.matmul(
        q.clamp_max(0), bound[:, :, 0].transpose(1, 2))
    score = score.amax(1)
    j = torch.arange(width, device="cuda")[None]
    blocks = ((s["lens"] + BLOCK - 1) // BLOCK)[:, None]
    score = torch.where((j < c["sink"]) | (j >= blocks - c["recent"]), math.inf, score)
    score = torch.where(j < blocks, score, -math.inf)
    n = min(n, width)
    best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :n]
    count = blocks[:, 0].clamp_max(n)
    best = torch.where(torch.arange(n, device="cuda")[None] < count[:, None], best, 1 << 30).sort(1).values
    picked = best < (1 << 30)
    at = torch.where(picked, best, 0)
    page, part = pages.gather(1, at // per), at % per
    k = s["kp"].view(-1, per, BLOCK, D)[page, part].float().view(rows, n * BLOCK, D)
    v = s["vp"].view(-1, per, BLOCK, D)[page, part].float().view(rows, n * BLOCK, D)
    pos = at[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    there = (picked[..., None] & (pos < s["lens"][:, None, None])).view(rows, 1, -1)
    p = _attend(torch.matmul(s["q"].float().view(rows, G, D), k.transpose(1, 2)) / math.sqrt(D), there)
    out = torch.matmul(p, v).view(b, heads, D).to(s["dtype"])
    listed_blocks = torch.full((rows, c["select"]), -1, dtype=torch.int32, device="cuda")
    listed_blocks[:, :n] = torch.where(picked, best, -1)
    return {"out": out, "blocks": listed_blocks, "counts": count.int()}


# ---- what a pass cannot do without

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    b, heads, kv = case["bsz"], case["heads"], case["kv"]
    lens, extra = _lengths(case)
    if case["op"] == "append":
        tokens = sum(extra)
        blocks = sum((n + extra[i // kv] - 1) // BLOCK - n // BLOCK + 1 for i, n in enumerate(lens))
        moved = tokens * D * e * (2 * heads + 4 * kv + 2) + (2 * blocks * 2 * D * e if case["bounds"] else 0)
        return {"bytes": moved + 12 * b * kv, "flops": 6 * tokens * D * (heads + kv)}
    io = 2 * b * heads * D * e
    if case["op"] == "shared":
        tokens = sum(extra) + sum(n - extra[i % kv] for i, n in enumerate(lens))
        return {"bytes": tokens * 2 * D * e + io, "flops": 4 * D * (heads // kv) * sum(lens)}
    blocks = [(n + BLOCK - 1) // BLOCK for n in lens]
    # all bounds, the keys and values of the chosen blocks
    taken = sum(min(n, BLOCK * min(case["select"], j)) for n, j in zip(lens, blocks))
    return {"bytes": sum(blocks) * 2 * D * e + taken * 2 * D * e + io + 4 * b * kv * case["select"],
            "flops": 2 * D * (heads // kv) * (2 * sum(blocks) + 2 * taken)}


# ---- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kv, heads, b = case["kv"], case["heads"], case["bsz"]
    lens, extra = _lengths(case)
    table = s["table"].tolist()
    if case["op"] == "append":
        cos, sin = s["cos"].double(), s["sin"].double()

        def turn(x):  # as the complex number x[d] + i x[d + 64] times c + i s, the two halves with their own tables
            x = x.double()
            a, z = x[..., :64], x[..., 64:]
            c, n = cos[:, None], sin[:, None]
            y = torch.empty_like(x)
            y[..., :64] = a * c[..., :64] - z * n[..., :64]
            y[..., 64:] = z * c[..., 64:] + a * n[..., 64:]
            return y
        q, k, v = turn(s["q"]), turn(s["k"]), s["v"].double()
        for i in range(b):
            q[i, :, extra[i]:] = 0
        kp, vp = s["kp"].double(), s["vp"].double()
        bounds = s["bounds"].double() if s["bounds"] is not None else None
        free, taken, ends = s["free"].tolist(), 0, []
        for i, n in enumerate(lens):
            end = n + extra[i // kv]
            ends.append(end)
            done = 0
            for p in range(n // PAGE, (end + PAGE - 1) // PAGE):
                if table[i][p] < 0:
                    table[i][p] = free[taken]
                    taken += 1
                page, lo, hi = table[i][p], max(n, p * PAGE), min(end, (p + 1) * PAGE)
                kp[page, lo - p * PAGE:hi - p * PAGE, 0] = k[i // kv, i % kv, done:done + hi - lo]
                vp[page, lo - p * PAGE:hi - p * PAGE, 0] = v[i // kv, i % kv, done:done + hi - lo]
                done += hi - lo
                if bounds is not None:
                    for u in range((lo - p * PAGE) // BLOCK, (hi - p * PAGE + BLOCK - 1) // BLOCK):
                        keys = kp[page, u * BLOCK:min((u + 1) * BLOCK, hi - p * PAGE), 0]
                        bounds[page, u, 0], bounds[page, u, 1] = keys.min(0).values, keys.max(0).values
        got = dict(q_out=q, kp=kp, vp=vp, table=_cuda(table), lens_out=_cuda(ends), free_ptr=_cuda([taken]))
        if bounds is not None:
            got["bounds"] = bounds
        return got
    G = heads // kv
    q = s["q"].double().view(b, kv, G, D)
    out = torch.zeros(b, kv, G, D, dtype=torch.float64, device="cuda")
    chosen = torch.full((b * kv, case.get("select", 0)), -1, dtype=torch.int64)
    for i, n in enumerate(lens):
        h = i % kv
        ids = list(table[i])
        if case["op"] == "shared":  # the first sequence's pages hold the shared tokens
            m = extra[h]
            where = torch.arange(n, device="cuda")
            first, mine = _cuda(table[h], torch.int64), _cuda(ids, torch.int64)
            page = torch.where(where < m, first[where // PAGE], mine[where // PAGE])
            k, v = s["kp"][page, where % PAGE, 0].double(), s["vp"][page, where % PAGE, 0].double()
        else:
            m = (n + BLOCK - 1) // BLOCK
            pages = _cuda(ids, torch.int64)
            blk = torch.arange(m, device="cuda")
            lim = s["bounds"][pages[blk // 4], blk % 4].double()
            lo, hi = lim[:, 0], lim[:, 1]
            u = torch.stack([torch.maximum(x * lo, x * hi).sum(1) for x in q[i // kv, h]]).amax(0).cpu().tolist()
            must = [x for x in range(m) if x < case["sink"] or x >= m - case["recent"]]
            rest = sorted((x for x in range(m) if x not in set(must)), key=lambda x: (-u[x], x))
            pick = sorted((must + rest)[:case["select"]])
            chosen[i, :len(pick)] = torch.tensor(pick)
            where = (_cuda(pick, torch.int64)[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten()
            where = where[where < n]
            page = pages[where // PAGE]
            k, v = s["kp"][page, where % PAGE, 0].double(), s["vp"][page, where % PAGE, 0].double()
        w = torch.softmax(q[i // kv, h] @ k.T * D ** -0.5, -1)
        out[i // kv, h] = w @ v
    out = out.view(b, heads, D)
    if case["op"] == "shared":
        return out
    return {"out": out, "blocks": chosen.int().cuda(), "counts": (chosen >= 0).sum(1).int().cuda()}
