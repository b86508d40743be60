"""The paged K/V cache: attention over it, for single tokens and for chunks of new tokens, and the management of its pages.

`own` False: the plain forms, elementary torch operations in 32 bits.  `own` True: the calls a program makes of the
library (allpaka_amd.Backend, allpaka_amd.PagedCache).  K and V are fp16 planes [capacity, n_kv * head_dim]; page p is
the rows [p * page, (p + 1) * page) of both; key j of sequence s is row table[s][j // page] * page + j % page.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # a chat of one user on a small model: the smallest call, bound by launches (16 query heads on 8, f32 activations)
        dict(name="decode_one_short", op="decode", n_seq=1, lo=600, hi=600, n_q=16, n_kv=8, hd=128, page=16, dtype="f32", window=0),
        # one user with a long document: one row per kv head over 128 Ki keys, split over the whole chip
        dict(name="decode_one_long", op="decode", n_seq=1, lo=131071, hi=131071, n_q=64, n_kv=8, hd=128, page=64, dtype="f16", window=0),
        # the decode step of a busy server: 64 requests of very different lengths
        dict(name="decode_batch", op="decode", n_seq=64, lo=100, hi=12000, n_q=64, n_kv=8, hd=128, page=16, dtype="f16", window=0),
        # heads of 64 in odd groups of 7 on odd pages, a sliding window, f32 activations
        dict(name="decode_odd_window", op="decode", n_seq=37, lo=3, hi=9001, n_q=14, n_kv=2, hd=64, page=23, dtype="f32", window=4096),
        # speculative decoding: a handful of draft tokens of each request verified at once
        dict(name="verify_drafts", op="chunk", n_seq=16, new_lo=1, new_hi=7, lo=500, hi=8000, n_q=64, n_kv=8, hd=128, page=16, dtype="f16", window=0),
        # the first chunk of one prompt: causal, nothing cached yet
        dict(name="prefill_first", op="chunk", n_seq=1, new_lo=2048, new_hi=2048, lo=0, hi=0, n_q=64, n_kv=8, hd=128, page=64, dtype="f16", window=0),
        # a later chunk of a long prompt over what is cached
        dict(name="chunk_long", op="chunk", n_seq=1, new_lo=512, new_hi=512, lo=32000, hi=32000, n_q=64, n_kv=8, hd=128, page=64, dtype="f16", window=0),
        # a mixed batch: single tokens and chunks together, f32 activations, heads of 64, a window
        dict(name="chunk_mixed_f32", op="chunk", n_seq=24, new_lo=1, new_hi=700, lo=0, hi=5000, n_q=16, n_kv=4, hd=64, page=24, dtype="f32", window=2000),
        # wide heads, several prompts of odd lengths
        dict(name="prefill_wide", op="chunk", n_seq=5, new_lo=333, new_hi=2500, lo=0, hi=1500, n_q=16, n_kv=4, hd=256, page=32, dtype="f16", window=0),
        # every decode step of a server: a row for each request, a few of them on pages they still share
        dict(name="pages_step", op="step", n_seq=256, lo=10, hi=1500, new=1, beams=8, planes=16, n_kv=8, hd=128, page=16),
        # a parallel sampling request arrives: its prompt forked, others freed, all extended, the shared tails copied
        dict(name="pages_fork", op="fork", n_seq=96, lo=10, hi=800, new=3, beams=32, planes=64, n_kv=8, hd=128, page=33),
        # a fragmented pool closed up: half of its requests freed, the rest moved to the front
        dict(name="pages_compact", op="compact", n_seq=128, lo=10, hi=700, moves=600, planes=32, n_kv=8, hd=128, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 3e14 + 2e-6


_LARGEST = {}


def draw(rng):
    if not _LARGEST:
        for c in listed():
            kind = c["op"] if c["op"] in ("decode", "chunk") else "pages"
            _LARGEST[kind] = max(_LARGEST.get(kind, 0.0), _cost(c))
    while True:
        kind = rng.choice(["decode", "decode", "chunk", "chunk", "chunk", "pages"])
        if kind == "pages":
            op = rng.choice(["step", "fork", "compact"])
            c = dict(op=op, n_seq=_log(rng, 2, 300), lo=rng.randint(1, 60), hi=_log(rng, 61, 3000), planes=2 * rng.randint(1, 32),
                     n_kv=rng.choice([1, 2, 4, 8]), hd=rng.choice([64, 128]), page=rng.choice([8, 16, 16, 32, 64, rng.randint(1, 100)]))
            if op == "compact":
                c["moves"] = rng.randint(1, 400)
            else:
                c["new"] = rng.randint(1, 20)
                c["beams"] = rng.randint(1, max(1, c["n_seq"] - 1))
            if _region_bytes(c) > 4 << 30:
                continue
        else:
            hd = rng.choice([64, 128, 128, 128, 256])
            n_kv = rng.choice([1, 2, 4, 8, 8])
            c = dict(op=kind, n_seq=_log(rng, 1, 200), lo=0, hi=0, n_q=n_kv * rng.choice([1, 2, 4, 5, 7, 8, 8, 16]), n_kv=n_kv, hd=hd,
                     page=rng.choice([16, 16, 32, 64, 128, rng.randint(1, 200)]), dtype=rng.choice(["f16", "f16", "f32"]),
                     window=rng.choice([0, 0, 0, _log(rng, 1, 5000)]))
            c["hi"] = _log(rng, 1, 131072) if kind == "decode" else rng.choice([0, _log(rng, 1, 40000)])
            c["lo"] = rng.randint(min(1, c["hi"]), c["hi"])
            if kind == "chunk":
                c["new_hi"] = _log(rng, 1, 4000)
                c["new_lo"] = rng.randint(1, c["new_hi"])
        if _cost(c) <= _LARGEST[kind]:
            return c


# Lengths follow from the case alone (the seed only orders them), so that work() is what every seed computes.
def _spread(n, lo, hi):
    return [lo + int((hi - lo) * (((i + 1) * 0.6180339887498949) % 1.0) + 0.5) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """(cached tokens, new tokens) of every sequence of an attention case; a single token's own key counts as new"""
    if case["op"] == "decode":
        return [(max(n, 1) - 1, 1) for n in _spread(case["n_seq"], case["lo"], case["hi"])]
    past = _spread(case["n_seq"], case["lo"], case["hi"])
    new = _spread(case["n_seq"] + 3, case["new_lo"], case["new_hi"])[3:]
    return list(zip(past, new))


def _visible(past, new, window):
    """(pairs of a row and a key it sees, keys that any row sees) of one sequence"""
    if not window:
        return new * past + new * (new + 1) // 2, past + new
    n = sum(min(window, past + r + 1) for r in range(new))
    return n, past + new - max(0, past + 1 - window)


def work(case):
    if case["op"] in ("decode", "chunk"):
        nq, nkv, hd = case["n_q"], case["n_kv"], case["hd"]
        es = 4 if case["dtype"] == "f32" else 2
        pairs = keys = rows = 0
        for past, new in _lens(case):
            a, b = _visible(past, new, case["window"])
            pairs, keys, rows = pairs + a, keys + b, rows + new
        return {"bytes": float(keys * nkv * hd * 2 * 2 + 2 * rows * nq * hd * es + 4 * (keys // case["page"] + 2 * case["n_seq"])),
                "flops": float(4 * hd * nq * pairs)}
    copied, words = _page_counts(case)
    return {"bytes": float(2 * copied * case["planes"] * _page_bytes(case) + 4 * words), "flops": 0.0}


# ------------------------------------------------------------------------------------------------- attention


def _rng(seed):
    return np.random.default_rng([0xCAC4E, int(seed)])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    return _prepare_attention(case, seed) if case["op"] in ("decode", "chunk") else _prepare_pages(case, seed)


def _prepare_attention(case, seed):
    r = _rng(seed)
    P, nkv, hd = case["page"], case["n_kv"], case["hd"]
    lens = [_lens(case)[i] for i in r.permutation(case["n_seq"])]
    counts = [_ceil(past + new, P) for past, new in lens]
    n_pages = sum(counts) + 3  # a few pages belong to nobody
    order = r.permutation(n_pages)
    width = max(counts) + 2
    table = np.full((len(lens), width), -1, np.int32)  # entries that no key needs hold anything
    at, used = 0, np.zeros(n_pages * P, bool)
    for s, (c, (past, new)) in enumerate(zip(counts, lens)):
        table[s, :c] = order[at:at + c]
        at += c
        rows = (table[s, :c].astype(np.int64)[:, None] * P + np.arange(P)).reshape(-1)[:past + new]
        used[rows] = True
    g = _gen(seed)
    planes = []
    unused = torch.from_numpy(~used).cuda()
    for _ in range(2):
        t = torch.empty((n_pages * P, nkv * hd), dtype=torch.float16, device="cuda").normal_(generator=g)
        t[unused] = float("nan")  # rows that were never written hold anything
        planes.append(t)
    q_off = np.concatenate([[0], np.cumsum([new for _, new in lens])])
    rows = int(q_off[-1])
    dt = DTYPES[case["dtype"]]
    q = torch.empty((rows, case["n_q"] * hd), dtype=torch.float32, device="cuda").normal_(generator=g).mul_(1.5).to(dt)
    state = dict(case=case, q=q, k=planes[0], v=planes[1], table=_i32(table), kv_len=_i32([a + b for a, b in lens]), q_off=_i32(q_off),
                 lens=lens, scale=1.0 / math.sqrt(hd), out=torch.empty_like(q))
    if own:
        state["be"] = _backend()
    return state


_be = []


def _backend():
    if not _be:
        import allpaka_amd

        _be.append(allpaka_amd.Backend(0))
    return _be[0]


def run(s):
    c = s["case"]
    if c["op"] in ("decode", "chunk"):
        if own:
            heads = (c["n_q"], c["n_kv"], c["hd"], s["scale"])
            if c["op"] == "decode":
                s["be"].attend_paged_into(s["q"], s["k"], s["v"], c["page"], s["table"], s["kv_len"], *heads, s["out"], window=c["window"])
            else:
                s["be"].attend_paged_chunk_into(s["q"], s["k"], s["v"], c["page"], s["table"], s["q_off"], s["kv_len"], *heads, s["out"], window=c["window"])
            return s["out"]
        return _plain_attention(s)
    return _own_pages(s) if own else _plain_pages(s)


def _plain_attention(s):
    """Sequence by sequence: its pages gathered, scores, mask, softmax, the weighted sum of the values."""
    c = s["case"]
    P, nq, nkv, hd, window = c["page"], c["n_q"], c["n_kv"], c["hd"], c["window"]
    out = torch.empty(s["q"].shape, dtype=torch.float32, device="cuda")
    block = max(1, (1 << 27) // max(1, max(a + b for a, b in s["lens"]) * nq))  # rows whose scores are held at once
    at = 0
    for i, (past, new) in enumerate(s["lens"]):
        n = past + new
        slots = (s["table"][i, :_ceil(n, P)].long()[:, None] * P + torch.arange(P, device="cuda")).reshape(-1)[:n]
        K = s["k"][slots].float().view(n, nkv, hd).permute(1, 2, 0).contiguous()
        V = s["v"][slots].float().view(n, nkv, hd).permute(1, 0, 2).contiguous()
        for r0 in range(0, new, block):
            r1 = min(new, r0 + block)
            m = r1 - r0
            q = s["q"][at + r0:at + r1].float().view(m, nkv, nq // nkv, hd).permute(1, 0, 2, 3).reshape(nkv, -1, hd)
            x = torch.matmul(q, K).view(nkv, m, nq // nkv, n) * s["scale"]
            if new > 1 or window:
                p = torch.arange(past + r0, past + r1, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None, :]
                hide = j > p
                if window:
                    hide = hide | (j <= p - window)
                x = x.masked_fill(hide[None, :, None, :], float("-inf"))
            e = torch.exp(x - x.max(dim=-1, keepdim=True).values)
            o = torch.matmul(e.view(nkv, -1, n), V).view(nkv, m, nq // nkv, hd) / e.sum(dim=-1, keepdim=True)
            out[at + r0:at + r1] = o.permute(1, 0, 2, 3).reshape(m, -1)
        at += new
    return out.to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- pages


def _page_bytes(c):
    return c["page"] * c["n_kv"] * c["hd"] * 2


def _layout(c):
    """Lengths and counts of a page case: what follows from the case alone."""
    P = c["page"]
    lens = _spread(c["n_seq"], c["lo"], c["hi"])
    d = dict(lens=lens, pages=[_ceil(n, P) for n in lens])
    if c["op"] == "step":  # sequence 0's prompt is shared by the next beams - 1 sequences, its unfull last page too
        d["beams"] = min(c["beams"], c["n_seq"])
        d["lens"] = lens = [lens[0]] * d["beams"] + lens[d["beams"]:]
        d["pages"] = [_ceil(n, P) for n in lens]
        d["live"] = sum(d["pages"]) - (d["beams"] - 1) * d["pages"][0]
        d["width"] = max(_ceil(n + c["new"], P) for n in lens) + 1
        d["n_pages"] = d["live"] + c["n_seq"] * (c["new"] // P + 2) + 5
    elif c["op"] == "fork":  # the last `beams` sequences are freed and become forks of sequence 0
        d["beams"] = min(c["beams"], c["n_seq"] - 1)
        d["live"] = sum(d["pages"])
        d["width"] = max(_ceil(n + c["new"], P) for n in lens) + 1
        d["n_pages"] = d["live"] + c["n_seq"] * (c["new"] // P + 2) + 5
    else:  # the second half of the sequences is freed; `moves` of the pages that stay lie behind where they shall
        d["keep"] = c["n_seq"] - c["n_seq"] // 2
        d["kept"] = sum(d["pages"][:d["keep"]])
        d["moves"] = min(c["moves"], d["kept"])
        d["live"] = sum(d["pages"])
        d["n_pages"] = d["live"] + d["moves"] + 5
        d["width"] = max(d["pages"]) + 1
    return d


def _region_bytes(c):
    return _layout(c)["n_pages"] * _page_bytes(c) * c["planes"]


def _page_counts(c):
    """(pages copied, words of metadata that have to be read or written)"""
    d, P = _layout(c), c["page"]
    if c["op"] == "compact":
        return d["moves"], 2 * d["n_pages"] + 2 * d["kept"]
    n0 = d["lens"][0]
    shared = d["beams"] - 1 if c["op"] == "step" else d["beams"]
    copied = shared if n0 % P else 0
    words = 2 * d["n_pages"] + c["n_seq"] * (4 + 2 * c["new"]) + (2 * d["beams"] * d["pages"][0] if c["op"] == "fork" else 0)
    return copied, words


def _prepare_pages(case, seed):
    r = _rng(seed)
    d = _layout(case)
    P, n_seq, n_pages = case["page"], case["n_seq"], d["n_pages"]
    table = np.full((n_seq, d["width"]), -1, np.int32)
    if case["op"] == "compact":
        # exactly `moves` kept pages at or behind index kept; the freed sequences' pages anywhere else
        low, high = r.permutation(d["kept"]), d["kept"] + r.permutation(n_pages - d["kept"])
        keep = r.permutation(np.concatenate([low[:d["kept"] - d["moves"]], high[:d["moves"]]]))
        rest = r.permutation(np.concatenate([low[d["kept"] - d["moves"]:], high[d["moves"]:]]))
        order = np.concatenate([keep, rest])
    else:
        order = r.permutation(n_pages)
    at = 0
    for s in range(n_seq):
        if case["op"] == "step" and 0 < s < d["beams"]:
            table[s] = table[0]
            continue
        table[s, :d["pages"][s]] = order[at:at + d["pages"][s]]
        at += d["pages"][s]
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    region = torch.empty((case["planes"], n_pages * P, case["n_kv"] * case["hd"]), dtype=torch.float16, device="cuda").normal_(generator=_gen(seed))
    state = dict(case=case, d=d, region=region, table0=_i32(table), refs0=_i32(refs), len0=_i32(d["lens"]))
    state["new"] = _i32(np.full(n_seq, case.get("new", 0)))
    if case["op"] == "fork":
        b = d["beams"]
        cut = np.full(n_seq, -1)
        cut[n_seq - b:] = 0
        state["cut"], state["src"], state["dst"] = _i32(cut), _i32(np.zeros(b)), _i32(np.arange(n_seq - b, n_seq))
    if case["op"] == "compact":
        state["cut"] = _i32(np.where(np.arange(n_seq) < d["keep"], -1, 0))
    if own:
        import allpaka_amd

        cache = allpaka_amd.PagedCache(_backend(), region, P, n_seq, d["width"])
        cache.adopt(state["table0"], state["len0"])
        state["cache"], state["saved"] = cache, cache.save()
    return state


def _own_pages(s):
    """Every pass begins from the same tables (a copy of three small arrays); the pages moved stay where they came from too."""
    c, cache = s["case"], s["cache"]
    cache.restore(s["saved"])
    if c["op"] == "compact":
        cache.truncate(s["cut"])
        cache.compact()
        return [cache.page_table, cache.kv_len, cache.refs, s["region"]]
    if c["op"] == "fork":
        cache.truncate(s["cut"])
        cache.fork(s["src"], s["dst"])
    step = cache.extend(s["new"], c["n_seq"] * c["new"])
    return [cache.page_table, cache.kv_len, cache.refs, step.q_off, step.positions, step.slots, s["region"]]


def _plain_pages(s):
    c, P = s["case"], s["case"]["page"]
    table, refs, lens = s["table0"].long(), s["refs0"].long(), s["len0"].long()
    n_seq, width = table.shape
    n_pages = refs.numel()
    col = torch.arange(width, device="cuda")
    pages = s["region"].view(c["planes"], n_pages, -1)

    def i32(*ts):
        return [t.to(torch.int32) for t in ts]

    if c["op"] != "step":  # pages past the new length lose a reference
        cut = torch.where(s["cut"].long() < 0, lens, torch.minimum(lens, s["cut"].long()))
        gone = (col >= ((cut + P - 1) // P)[:, None]) & (col < ((lens + P - 1) // P)[:, None])
        refs = refs - torch.bincount(table[gone], minlength=n_pages)
        lens = cut
    if c["op"] == "compact":
        live = refs > 0
        n = int(live.sum())
        idx = torch.arange(n_pages, device="cuda")
        src, dst = idx[live & (idx >= n)], idx[~live & (idx < n)]
        pages[:, dst] = pages[:, src]
        name = idx.clone()
        name[src] = dst
        inside = col < ((lens + P - 1) // P)[:, None]
        table[inside] = name[table[inside]]
        refs[dst] = refs[src]
        refs[src] = 0
        return i32(table, lens, refs) + [s["region"]]
    if c["op"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        inside = col < ((lens[src] + P - 1) // P)[:, None]
        table[dst] = torch.where(inside, table[src], table[dst])
        refs = refs + torch.bincount(table[src][inside], minlength=n_pages)
        lens[dst] = lens[src]
    new = s["new"].long()
    have, want = (lens + P - 1) // P, (lens + new + P - 1) // P
    tail = torch.where((lens % P != 0) & (new > 0), table[torch.arange(n_seq, device="cuda"), (lens // P).clamp(max=width - 1)], -1)
    held = torch.where(tail >= 0, refs[tail.clamp(min=0)], 0)
    seqs = torch.arange(n_seq, device="cuda")
    # of the holders of an unfull page that all write now the last one keeps it, the others write to a copy
    count = torch.bincount(tail[tail >= 0], minlength=n_pages)[tail.clamp(min=0)]
    last = torch.zeros(n_pages, dtype=torch.long, device="cuda").scatter_reduce_(0, tail.clamp(min=0), torch.where(tail >= 0, seqs, -1), "amax")[tail.clamp(min=0)]
    copies = (held > 1) & ~((count == held) & (last == seqs))
    need = want - have + copies.long()
    free = torch.nonzero(refs == 0).view(-1)
    first = torch.cumsum(need, 0) - need
    src, dst = tail[copies], free[first[copies]]
    pages[:, dst] = pages[:, src]
    refs = refs - torch.bincount(src, minlength=n_pages)
    table[seqs[copies], (lens // P)[copies]] = dst
    fresh = (col >= have[:, None]) & (col < want[:, None])
    table = torch.where(fresh, free[((first + copies.long())[:, None] + col - have[:, None]).clamp(0, free.numel() - 1)], table)
    refs[free[:int(need.sum())]] = 1
    lens2 = lens + new
    q_off = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(new, 0)])
    row = torch.arange(int(q_off[-1]), device="cuda")
    of = torch.searchsorted(q_off, row, right=True) - 1
    positions = lens[of] + row - q_off[of]
    slots = table[of, positions // P] * P + positions % P
    return i32(table, lens2, refs, q_off, positions, slots) + [s["region"]]


# ------------------------------------------------------------------------------------------------- from the definitions


def exact(case, seed):
    return _exact_attention(case, seed) if case["op"] in ("decode", "chunk") else _exact_pages(case, seed)


def _exact_attention(case, seed):
    """Head by head in 64 bits: logits, their log-sum-exp, the expectation of the values."""
    s = _prepare_attention(case, seed)
    P, nq, nkv, hd, window = case["page"], case["n_q"], case["n_kv"], case["hd"], case["window"]
    if work(case)["flops"] > 2e13:
        return None
    q = s["q"].double().view(-1, nq, hd)
    out = torch.zeros_like(q)
    q_off, kv_len, table = s["q_off"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    for i, n in enumerate(kv_len):
        a, b = q_off[i], q_off[i + 1]
        where = torch.tensor([table[i][j // P] * P + j % P for j in range(n)], device="cuda")
        k, v = (t.index_select(0, where).double() for t in (s["k"], s["v"]))
        step = max(1, (1 << 26) // n)
        for h in range(nq):
            lane = slice(h // (nq // nkv) * hd, (h // (nq // nkv) + 1) * hd)
            kh, vh = k[:, lane].t().contiguous(), v[:, lane].contiguous()
            for r in range(a, b, step):
                e = min(b, r + step)
                z = torch.mm(q[r:e, h].contiguous(), kh) * s["scale"]
                pos = torch.arange(n - (b - r), n - (b - e), device="cuda")
                key = torch.arange(n, device="cuda")
                seen = key[None] <= pos[:, None]
                if window:
                    seen &= key[None] + window > pos[:, None]
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                out[r:e, h] = torch.mm(torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), vh)
    return out.view(-1, nq * hd)


def _exact_pages(case, seed):
    """One sequence after the other, page by page, with plain lists; then the pages, one by one."""
    s = _prepare_pages(case, seed)
    table, refs, lens = s["table0"].tolist(), s["refs0"].tolist(), s["len0"].tolist()
    cut, src, dst = (s[k].tolist() if k in s else [] for k in ("cut", "src", "dst"))
    pairs = []
    P, n_pages = case["page"], len(refs)
    if case["op"] != "step":
        for q, c in enumerate(cut):
            if 0 <= c < lens[q]:
                for i in range(_ceil(c, P), _ceil(lens[q], P)):
                    refs[table[q][i]] -= 1
                lens[q] = c
    if case["op"] == "compact":
        n = sum(x > 0 for x in refs)
        holes = [p for p in range(n) if refs[p] == 0]
        for p in range(n, n_pages):
            if refs[p]:
                to = holes.pop(0)
                pairs.append((to, p))
                refs[to], refs[p] = refs[p], 0
                for q in range(len(table)):
                    for i in range(_ceil(lens[q], P)):
                        if table[q][i] == p:
                            table[q][i] = to
        return [np.array(x, np.int32) for x in (table, lens, refs)] + [_moved(s, pairs)]
    for a, b in zip(src, dst):
        for i in range(_ceil(lens[a], P)):
            table[b][i] = table[a][i]
            refs[table[a][i]] += 1
        lens[b] = lens[a]
    q_off, positions, slots = [0], [], []
    free = iter([p for p in range(n_pages) if refs[p] == 0])
    for q in range(len(table)):
        new = case["new"]
        if lens[q] % P and refs[table[q][lens[q] // P]] > 1:
            refs[table[q][lens[q] // P]] -= 1
            old, p = table[q][lens[q] // P], next(free)
            pairs.append((p, old))
            table[q][lens[q] // P] = p
            refs[p] = 1
        for i in range(_ceil(lens[q], P), _ceil(lens[q] + new, P)):
            table[q][i] = p = next(free)
            refs[p] = 1
        for j in range(lens[q], lens[q] + new):
            positions.append(j)
            slots.append(table[q][j // P] * P + j % P)
        lens[q] += new
        q_off.append(q_off[-1] + new)
    return [np.array(x, np.int32) for x in (table, lens, refs, q_off, positions, slots)] + [_moved(s, pairs)]


def _moved(s, pairs):
    P = s["case"]["page"]
    for to, p in pairs:
        s["region"][:, to * P:(to + 1) * P].copy_(s["region"][:, p * P:(p + 1) * P])
    return s["region"]
