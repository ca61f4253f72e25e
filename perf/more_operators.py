"""The attention operators of a served model, over the sizes they are used at: causal attention over packed prompts, one
token over a paged cache of keys and values, the rows that new tokens take in it, and their storing.

With ``own`` false, ``run`` computes them in plain 32-bit torch (products, maxima, exponentials, sums, indexing) and
rounds once at the end; with ``own`` true it makes the calls of ``pto_fuser_amd`` that a program makes.  ``exact``
evaluates the definitions in 64 bits, sequence by sequence and head by head.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------
#  The cases
# ------------------------------------------------------------------------------------------
def _prefill(dtype, B, T, H, G, D=128, mix=0, padded=False):
    """B prompts of up to T tokens (all T where mix is 0), H query heads over G heads of keys and values, rows packed end
    to end or each prompt at a multiple of T."""
    return {"op": "prefill", "dtype": dtype, "B": B, "T": T, "H": H, "G": G, "D": D, "mix": mix, "padded": padded}


def _step(dtype, B, T, H, G, D=128, page=16, mix=0, pool=0):
    return {"op": "step", "dtype": dtype, "B": B, "T": T, "H": H, "G": G, "D": D, "page": page, "mix": mix, "pool": pool}


def _store(dtype, N, G, D=128, page=16):
    return {"op": "store", "dtype": dtype, "N": N, "G": G, "D": D, "page": page}


def _pages(kind, B, T, new, page=16, mix=1, pool=0, short=False):
    """kind 'assign': B requests with up to T tokens in the cache get up to ``new`` more each (``short``: from a pool with
    too few pages); 'release': they leave."""
    return {"op": "pages", "kind": kind, "B": B, "T": T, "new": new, "page": page, "mix": mix, "pool": pool, "short": short}


def listed():
    return [
        # the benchmark's prompts in an attention layer of its 16 heads, four of them to a head of keys
        dict(_prefill("bf16", 4, 4096, 16, 4), name="prefill_batch"),
        # one long context, 32 heads
        dict(_prefill("bf16", 1, 32768, 32, 8), name="prefill_long"),
        # 48 short prompts of uneven length, packed, one of them empty
        dict(_prefill("bf16", 48, 512, 16, 2, mix=7), name="prefill_chats"),
        # three prompts of uneven length in full precision, in a padded batch
        dict(_prefill("fp32", 3, 1471, 6, 2, D=64, mix=3, padded=True), name="prefill_ragged_fp32"),
        # one token each of 64 running sequences of uneven length
        dict(_step("bf16", 64, 8192, 16, 4, mix=5, pool=80), name="step_batch"),
        # one token of one long context
        dict(_step("bf16", 1, 131072, 32, 8, page=64), name="step_long"),
        # one token of one short sequence, a head of keys for each
        dict(_step("bf16", 1, 512, 4, 4), name="step_single"),
        # 24 sequences in full precision
        dict(_step("fp32", 24, 1471, 6, 2, D=64, page=32, mix=9), name="step_ragged_fp32"),
        # the keys and values of the benchmark's 16384 tokens, and of 64 single ones
        dict(_store("bf16", 16384, 4), name="store_prefill"),
        dict(_store("bf16", 64, 4), name="store_step"),
        # 64 prompts arrive; 256 running sequences grow by a token
        dict(_pages("assign", 64, 0, 1024, pool=96), name="pages_prefill"),
        dict(_pages("assign", 256, 8192, 1, pool=300), name="pages_step"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "prefill", "step", "step", "step", "store", "pages"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    mix = rng.choice([0, rng.randrange(1, 1 << 30)])
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    G = rng.choice([1, 2, 4, 8])
    H = G * rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "prefill":
        T = _log_int(rng, 1, 16384 if dtype == "bf16" else 4096)
        most = 4_000_000_000_000 if dtype == "bf16" else 250_000_000_000
        B = _log_int(rng, 1, max(1, min(64, int(most / (4.0 * D * H * T * (T + 1) / 2)), 60_000_000 // (T * (H + G) * D))))
        return _prefill(dtype, B, T, H, G, D, mix, padded=rng.random() < 0.3)
    if op == "step":
        most = 500_000_000 // (2 * ESIZE[dtype] * D * G)
        T = _log_int(rng, 1, min(131072, most))
        B = _log_int(rng, 1, max(1, min(256, most // T)))
        return _step(dtype, B, T, H, G, D, page, mix, pool=B + 3 if rng.random() < 0.5 else 0)
    if op == "store":
        return _store(dtype, _log_int(rng, 1, min(65536, 260_000_000 // (4 * ESIZE[dtype] * G * D))), G, D, page)
    kind, B = rng.choice(["assign", "assign", "release"]), _log_int(rng, 1, 1024)
    pool = B + 9 if rng.random() < 0.5 else 0
    if kind == "release":
        return _pages(kind, B, _log_int(rng, 1, 8192), 0, page, 1 + mix, pool)
    new = _log_int(rng, 1, max(1, min(8192, 65536 // B)))
    return _pages(kind, B, rng.choice([0, _log_int(rng, 1, 8192)]), new, page, 1 + mix, pool, short=rng.random() < 0.2)


def _lengths(case, B=None, T=None, key=0):
    """The sequences' lengths, from the case alone: all T, or uneven ones of 0 to T, the first whole and of three or more the
    last empty."""
    B, T = case["B"] if B is None else B, case["T"] if T is None else T
    if not case["mix"]:
        return [T] * B
    rng = random.Random(case["mix"] + key)
    n = [rng.randint(0, T) for _ in range(B)]
    n[0] = T
    if B > 2:
        n[-1] = 0
    return n


# ------------------------------------------------------------------------------------------
#  What a program has in hand before the call
# ------------------------------------------------------------------------------------------
def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return gen


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _perm(gen, n):
    return torch.randperm(n, generator=gen, device="cuda").to(torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _qkv(gen, rows, H, G, D, dt):
    """q, k, v [rows, heads, D] as views of one projected row a token.  Scores of unit queries and keys have a deviation of
    1; some keys are larger, as attention's sinks are."""
    row = _randn(gen, rows, (H + 2 * G) * D)
    row[::97, H * D:(H + G) * D] *= 3
    q, k, v = row.to(dt).split([H * D, G * D, G * D], dim=-1)
    return q.unflatten(-1, (H, D)), k.unflatten(-1, (G, D)), v.unflatten(-1, (G, D))


def _slots(gen, B, pool):
    return _perm(gen, pool)[:B].contiguous() if pool else None


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "prefill":
        n, B, T = _lengths(case), case["B"], case["T"]
        starts = [i * T for i in range(B + 1)] if case["padded"] else [sum(n[:i]) for i in range(B + 1)]
        s["q"], s["k"], s["v"] = _qkv(gen, starts[-1], case["H"], case["G"], case["D"], DTYPES[case["dtype"]])
        s["cu"], s["lengths"] = _ints(starts), _ints(n) if case["padded"] else None
        s["host"] = list(zip(starts, n))                 # a program that makes the batch knows its prompts
    elif op == "step":
        n, page, dt = _lengths(case), case["page"], DTYPES[case["dtype"]]
        need = [(x + page - 1) // page for x in n]
        width, pages = max(need) + 1, sum(need) + 5
        order = _perm(gen, pages)                        # pages in the order in which requests came by them
        table = torch.full((case["pool"] or case["B"], width), -1, dtype=torch.int32, device="cuda")
        s["slots"] = _slots(gen, case["B"], case["pool"])
        at = torch.arange(case["B"], device="cuda") if s["slots"] is None else s["slots"].long()
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        col = torch.arange(width, device="cuda")
        live = col < torch.tensor(need, device="cuda")[:, None]
        table[at] = torch.where(live, order[(first[:, None] + col).clamp(max=pages - 1)], -1)
        shape = (pages, page, case["G"], case["D"])
        s["k"], s["v"] = _randn(gen, *shape).to(dt), _randn(gen, *shape).to(dt)
        s["q"] = _randn(gen, case["B"], case["H"], case["D"]).to(dt)
        s["tables"], s["lengths"] = table, _ints(n)
    elif op == "store":
        N, G, D, page, dt = case["N"], case["G"], case["D"], case["page"], DTYPES[case["dtype"]]
        _, s["k"], s["v"] = _qkv(gen, N, G, G, D, dt)
        pages = (N + page - 1) // page + 3
        at = torch.arange(N, device="cuda")
        rows = _perm(gen, pages).long()[at // page] * page + at % page
        s["rows"] = torch.where(at % 61 == 60, -1, rows)          # tokens of requests that got no page
        s["k_cache"], s["v_cache"] = (_randn(gen, pages, page, G, D).to(dt) for _ in range(2))
    else:
        B, page = case["B"], case["page"]
        c = _lengths(case)
        n = [1] * B if case["new"] == 1 else _lengths(case, T=case["new"], key=1)
        have = [(x + page - 1) // page for x in c]
        want = [(x + y + page - 1) // page for x, y in zip(c, n)]
        grow, width = sum(want) - sum(have), max(want) + 1
        total = sum(have) + grow + 4
        order = _perm(gen, total)
        s["slots"] = _slots(gen, B, case["pool"])
        at = torch.arange(B, device="cuda") if s["slots"] is None else s["slots"].long()
        first = torch.tensor([sum(have[:i]) for i in range(B)], device="cuda")
        col = torch.arange(width, device="cuda")
        live = col < torch.tensor(have, device="cuda")[:, None]
        s["tables"] = torch.full((case["pool"] or B, width), -1, dtype=torch.int32, device="cuda")
        s["tables"][at] = torch.where(live, order[(first[:, None] + col).clamp(max=total - 1)], -1)
        s["free"] = order if not case["short"] else order[:sum(have) + max(grow // 2, 1)].contiguous()
        s["taken"] = _ints([sum(have)])
        s["lengths"], s["tokens"], s["capacity"] = _ints(c), _ints(n), sum(n) + 7
        if case["new"] == 1:
            s["capacity"] = B
    return s


# ------------------------------------------------------------------------------------------
#  One pass
# ------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    pf, case = _package(), s["case"]
    op = case["op"]
    if op == "prefill":
        return pf.causal_attention(s["q"], s["k"], s["v"], s["cu"], lengths=s["lengths"])
    if op == "step":
        return pf.attention_step(s["q"], s["k"], s["v"], s["tables"], s["lengths"], slots=s["slots"])
    if op == "store":
        pf.store_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["rows"])
        return s["k_cache"], s["v_cache"]
    if case["kind"] == "release":
        taken = pf.release_pages(s["tables"], s["lengths"], s["free"], s["taken"], page_size=case["page"], slots=s["slots"])
        return s["free"], taken
    plan = pf.assign_pages(s["tables"], s["lengths"], s["tokens"], s["free"], s["taken"], page_size=case["page"],
                           capacity=s["capacity"], slots=s["slots"])
    return plan.rows, plan.cu_seqlens, plan.lengths, plan.taken, s["tables"]


_PACKAGE = []


def _package():
    if not _PACKAGE:
        sys.path.insert(0, os.path.join(os.getcwd(), "pto-fuser_amd"))
        import pto_fuser_amd
        _PACKAGE.append(pto_fuser_amd)
    return _PACKAGE[0]


def _run_plain(s):
    op = s["case"]["op"]
    if op == "pages":
        return (_plain_release if s["case"]["kind"] == "release" else _plain_assign)(s)
    return {"prefill": _plain_prefill, "step": _plain_step, "store": _plain_store}[op](s)


def _plain_prefill(s):
    case = s["case"]
    H, G, D = case["H"], case["G"], case["D"]
    out = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    for start, n in s["host"]:
        if not n:
            continue
        q, k, v = (s[x][start:start + n].float() for x in "qkv")
        q = q.transpose(0, 1).reshape(G, H // G, n, D) * D ** -0.5
        k = k.permute(1, 2, 0).contiguous()[:, None]                   # [G, 1, D, n]
        v = v.transpose(0, 1).contiguous()[:, None]                    # [G, 1, n, D]
        rows = max(1, min(n, (1 << 27) // (H * n)))                    # of queries at a time
        for i in range(0, n, rows):
            j = min(i + rows, n)
            score = torch.matmul(q[:, :, i:j], k[..., :j])
            ahead = torch.arange(j, device=q.device) > torch.arange(i, j, device=q.device)[:, None]
            score = score.masked_fill_(ahead, -math.inf)
            p = score.sub_(score.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(p, v[:, :, :j]) / p.sum(-1, keepdim=True)
            out[start + i:start + j] = o.reshape(H, j - i, D).transpose(0, 1).to(out.dtype)
    return out


def _plain_step(s):
    case = s["case"]
    B, H, G, D, page = (case[k] for k in ("B", "H", "G", "D", "page"))
    table = s["tables"] if s["slots"] is None else s["tables"][s["slots"].long()]
    at, width = table.long().clamp(min=0), table.shape[1] * page
    k = s["k"][at].reshape(B, width, G, D).float().permute(0, 2, 3, 1).contiguous()      # [B, G, D, tokens]
    v = s["v"][at].reshape(B, width, G, D).float().transpose(1, 2).contiguous()
    score = torch.matmul(s["q"].float().reshape(B, G, H // G, D) * D ** -0.5, k)
    live = (torch.arange(width, device=score.device) < s["lengths"][:, None])[:, None, None]
    score = torch.where(live, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o.reshape(B, H, D).to(s["q"].dtype)


def _plain_store(s):
    keep = s["rows"] >= 0
    some = keep.int().argmax()                            # a token without a row repeats what one with a row writes
    at = torch.where(keep, s["rows"], s["rows"][some])
    for x in "kv":
        cache = s[x + "_cache"]
        cache.view(-1, *cache.shape[2:])[at] = torch.where(keep[:, None, None], s[x], s[x][some])
    return s["k_cache"], s["v_cache"]


def _ceil(n, page):
    return torch.div(n + page - 1, page, rounding_mode="floor")


def _plain_assign(s):
    page, cap, F = s["case"]["page"], s["capacity"], s["free"].shape[0]
    B, width = s["lengths"].shape[0], s["tables"].shape[1]
    dev = s["lengths"].device
    slots = torch.arange(B, device=dev) if s["slots"] is None else s["slots"].long()
    c, n, taken = s["lengths"].long(), s["tokens"].long(), s["taken"].long()
    end = n.cumsum(0)
    have, want = _ceil(c, page), _ceil(c + n, page)
    fits = (want <= width) & (end <= cap)
    need = torch.where(fits, want - have, 0)
    last = need.cumsum(0)
    served = fits & ((need == 0) | (taken + last <= F))
    cu = torch.nn.functional.pad(end, (1, 0)).clamp(max=cap)
    col = torch.arange(width, device=dev)
    old = s["tables"][slots]
    fresh = s["free"][(taken + (last - need)[:, None] + col - have[:, None]).clamp(0, F - 1)]
    new = torch.where(served[:, None] & (col >= have[:, None]) & (col < want[:, None]), fresh, old)
    s["tables"][slots] = new
    t = torch.arange(cap, device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = b < B
    b = b.clamp(max=B - 1)
    at = c[b] + t - cu[b]
    entry = new[b, (at // page).clamp(max=width - 1)].long()
    rows = torch.where(live & served[b], entry * page + at % page, -1)
    lengths = torch.where(served, c + n, c)
    return rows, cu.int(), lengths.int(), (taken + torch.where(served, need, 0).sum()).int(), s["tables"]


def _plain_release(s):
    page, F = s["case"]["page"], s["free"].shape[0]
    slots = torch.arange(s["lengths"].shape[0], device=s["lengths"].device) if s["slots"] is None else s["slots"].long()
    n = _ceil(s["lengths"].long(), page)
    last, taken = n.cumsum(0), s["taken"].long()
    col = torch.arange(s["tables"].shape[1], device=n.device)
    put = torch.where(col < n[:, None], taken - 1 - ((last - n)[:, None] + col), F)
    free = torch.nn.functional.pad(s["free"], (0, 1)).scatter(0, put.flatten(), s["tables"][slots].flatten())
    s["free"].copy_(free[:F])
    return s["free"], (taken - last[-1:]).int()


# ------------------------------------------------------------------------------------------
#  What one pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    op, e = case["op"], ESIZE.get(case.get("dtype"), 4)
    if op == "prefill":
        n, H, G, D = _lengths(case), case["H"], case["G"], case["D"]
        return {"bytes": e * sum(n) * D * (2 * H + 2 * G), "flops": 4 * D * H * sum(x * (x + 1) // 2 for x in n)}
    if op == "step":
        n, H, G, D, page = _lengths(case), case["H"], case["G"], case["D"], case["page"]
        entries = sum((x + page - 1) // page for x in n)
        return {"bytes": 2 * e * sum(n) * G * D + 2 * e * case["B"] * H * D + 4 * entries, "flops": 4 * D * H * sum(n)}
    if op == "store":
        n = case["N"]
        return {"bytes": 4 * e * n * case["G"] * case["D"] + 8 * n, "flops": 0}
    B, page, c = case["B"], case["page"], _lengths(case)
    have = sum((x + page - 1) // page for x in c)
    if case["kind"] == "release":
        return {"bytes": 8 * B + 8 * have, "flops": 0}
    n = [1] * B if case["new"] == 1 else _lengths(case, T=case["new"], key=1)
    grow = sum((x + y + page - 1) // page for x, y in zip(c, n)) - have
    return {"bytes": 20 * B + 8 * grow + 8 * sum(n), "flops": 0}


# ------------------------------------------------------------------------------------------
#  The definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "prefill":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for start, n in s["host"]:
            for h in range(case["H"] if n else 0):
                g = h * case["G"] // case["H"]
                q, k, v = s["q"][start:start + n, h].double(), s["k"][start:start + n, g].double(), s["v"][start:start + n, g].double()
                for i in range(0, n, 4096):
                    j = min(i + 4096, n)
                    score = q[i:j] @ k[:j].t().contiguous() / math.sqrt(case["D"])
                    score += torch.full_like(score, -math.inf).triu(i + 1)
                    out[start + i:start + j, h] = torch.softmax(score, -1) @ v[:j]
        return out
    if op == "step":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            if not n:
                continue
            row = s["tables"][b if s["slots"] is None else int(s["slots"][b])]
            pages = row[:(n + case["page"] - 1) // case["page"]].long()
            k, v = (s[x][pages].flatten(0, 1)[:n].double() for x in "kv")
            for h in range(case["H"]):
                g = h // (case["H"] // case["G"])
                w = torch.softmax((k[:, g] * s["q"][b, h].double()).sum(-1) / math.sqrt(case["D"]), 0)
                out[b, h] = (w[:, None] * v[:, g]).sum(0)
        return out
    if op == "store":
        for t, r in enumerate(s["rows"].tolist() if case["N"] <= 64 else []):
            if r >= 0:
                s["k_cache"][r // case["page"], r % case["page"]] = s["k"][t]
                s["v_cache"][r // case["page"], r % case["page"]] = s["v"][t]
        if case["N"] > 64:
            keep = torch.nonzero(s["rows"] >= 0)[:, 0]
            r = s["rows"][keep]
            s["k_cache"][r // case["page"], r % case["page"]] = s["k"][keep]
            s["v_cache"][r // case["page"], r % case["page"]] = s["v"][keep]
        return s["k_cache"].double(), s["v_cache"].double()
    return None
