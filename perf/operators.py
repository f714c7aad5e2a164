"""Workloads of the serving operators: packed prompt attention, the 4-bit paged cache (store, load, one-token
attention) and the cache's page bookkeeping.  Each case runs in a plain form (elementary torch operations in fp32) or,
with `own`, through the framework's launch graph."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# --------------------------------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # Four chat turns of a few dozen tokens arriving together: a call bound by latency.
        prompt("prompt_turns", seqs=4, longest=61, hq=32, hkv=8, dim=128, dtype="bfloat16"),
        # A prefill batch of prompts from one token to a page of text, packed from one fused projection.
        prompt("prompt_mixed", seqs=16, longest=1021, hq=32, hkv=8, dim=128, dtype="bfloat16"),
        # One long document through the attention heads of the decoder layer this repository measures.
        prompt("prompt_document", seqs=1, longest=8192, hq=32, hkv=8, dim=128, dtype="bfloat16"),
        # Chunks of prompts whose prefixes were cached earlier (queries see more keys than there are queries), small heads.
        prompt("prompt_prefixed_d64", seqs=12, longest=700, hq=16, hkv=2, dim=64, dtype="float16", prefix=1500),
        # One chat with a few hundred tokens of context: a decode step bound by latency.
        decode("decode_chat", slots=1, longest=700, hq=32, hkv=8, dim=128, page=16, group=64, dtype="bfloat16"),
        # A serving batch at ragged depths, from fresh requests to 8k of context.
        decode("decode_batch", slots=64, longest=8191, hq=32, hkv=8, dim=128, page=16, group=64, dtype="bfloat16"),
        # Few requests with book-length context.
        decode("decode_book", slots=4, longest=131072, hq=32, hkv=8, dim=128, page=64, group=64, dtype="bfloat16"),
        # Small heads, many query heads per cached head, finer groups, the other 16-bit type.
        decode("decode_d64", slots=33, longest=5000, hq=32, hkv=2, dim=64, page=32, group=32, dtype="float16"),
        # The K and V of one decode step of a batch written to the cache and read back.
        store("store_step", slots=64, longest=1, context=2000, hkv=8, dim=128, page=16, group=64, dtype="bfloat16"),
        # The K and V of a prefill batch written to the cache and read back.
        store("store_prompts", slots=24, longest=2047, context=300, hkv=8, dim=128, page=16, group=64, dtype="bfloat16"),
        # A sampling step that replaces half of the slots by forks of the others.
        pages("pages_fork", act="fork", slots=64, longest=4000, hkv=8, dim=128, page=16, group=64, layers=2),
        # Half of the requests leave, the cache is compacted, new requests take their pages.
        pages("pages_turnover", act="turnover", slots=48, longest=1500, hkv=8, dim=128, page=16, group=64, layers=4),
    ]


def prompt(name=None, *, seqs, longest, hq, hkv, dim, dtype, prefix=0):
    return named(name, op="prompt", seqs=seqs, longest=longest, hq=hq, hkv=hkv, dim=dim, dtype=dtype, prefix=prefix)


def decode(name=None, *, slots, longest, hq, hkv, dim, page, group, dtype):
    return named(name, op="decode", slots=slots, longest=longest, hq=hq, hkv=hkv, dim=dim, page=page, group=group,
                 dtype=dtype)


def store(name=None, *, slots, longest, context, hkv, dim, page, group, dtype):
    return named(name, op="store", slots=slots, longest=longest, context=context, hkv=hkv, dim=dim, page=page,
                 group=group, dtype=dtype)


def pages(name=None, *, act, slots, longest, hkv, dim, page, group, layers):
    return named(name, op="pages", act=act, slots=slots, longest=longest, hkv=hkv, dim=dim, page=page, group=group,
                 layers=layers)


def named(name, **case):
    return case if name is None else dict(case, name=name)


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["prompt", "prompt", "decode", "decode", "store", "pages"])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    page = rng.choice([16, 32, 64, 128])
    if op == "prompt":
        per = rng.choice([1, 3, 4, 8])
        longest, hq = spread(1, 4096), hkv * per
        most = max(1, min(64, (1 << 31) // (hq * longest * longest * 2)))
        prefix = rng.choice([0, 0, spread(1, 2048)]) if longest <= 2048 else 0
        if prefix:
            most = max(1, most * longest // (longest + prefix))
        return prompt(seqs=spread(1, most), longest=longest, hq=hq, hkv=hkv, dim=dim, dtype=dtype, prefix=prefix)
    if op == "decode":
        per = rng.choice([1, 3, 4, 8, 16])
        longest = spread(1, 65536)
        slots = spread(1, max(1, min(256, (1 << 21) // (hkv * longest))))
        return decode(slots=slots, longest=longest, hq=hkv * per, hkv=hkv, dim=dim, page=page, group=group, dtype=dtype)
    if op == "store":
        longest = spread(1, 4096)
        slots = spread(1, max(1, min(128, 49152 // longest)))
        return store(slots=slots, longest=longest, context=spread(1, 4096), hkv=hkv, dim=dim, page=page, group=group,
                     dtype=dtype)
    longest = spread(1, 4096)
    slots = spread(4, max(4, min(128, 65536 // longest)))
    return pages(act=rng.choice(["fork", "copy", "turnover"]), slots=slots, longest=longest, hkv=hkv, dim=dim, page=page,
                 group=group, layers=rng.choice([1, 2, 3]))


def lengths(case, count, longest, salt=0):
    """`count` lengths in 1..longest, one of them `longest`: what a batch of requests holds, the same for every seed."""
    rng = random.Random("%d %d %d" % (count, longest, salt))
    out = [max(1, int(round(longest * rng.random() ** 1.5))) for _ in range(count)]
    out[rng.randrange(count)] = longest
    return out


def prompt_lengths(case):
    ql = lengths(case, case["seqs"], case["longest"])
    pre = [0] * case["seqs"]
    if case["prefix"]:
        pre = [p - 1 for p in lengths(case, case["seqs"], case["prefix"] + 1, 1)]
    return ql, [a + b for a, b in zip(ql, pre)]


def page_bytes(case):
    return case["hkv"] * case["page"] * (case["dim"] + 8 * (case["dim"] // case["group"]))


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def work(case):
    op, d = case["op"], case["dim"]
    if op == "prompt":
        ql, kl = prompt_lengths(case)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(ql, kl))
        return {"bytes": 4 * d * (case["hq"] * sum(ql) + case["hkv"] * sum(kl)), "flops": 4 * d * case["hq"] * pairs}
    if op == "decode":
        total = sum(lengths(case, case["slots"], case["longest"]))
        return {"bytes": total * page_bytes(case) // case["page"] + 4 * case["slots"] * case["hq"] * d,
                "flops": 4 * total * case["hq"] * d}
    if op == "store":
        total = sum(lengths(case, case["slots"], case["longest"]))
        return {"bytes": total * (8 * case["hkv"] * d + page_bytes(case) // case["page"]), "flops": 12 * total * case["hkv"] * d}
    lens, table, refs, _ = page_state(case)
    return {"bytes": page_moves(case, lens, table) * 2 * case["layers"] * page_bytes(case), "flops": 0}


# --------------------------------------------------------------------------------------------------------------------
# The 4-bit page format: blocks of min(page, 32) tokens, in each [K codes | V codes | K params | V params]
# --------------------------------------------------------------------------------------------------------------------
def v_row(t):
    """Where a block keeps the V codes of its token t: in every eight, the even tokens first."""
    return (t & ~7) | ((t & 1) << 2) | ((t >> 1) & 3)


def k_bytes(code):
    """Codes [..., dim] of a key as its row of bytes."""
    w = code.unflatten(-1, (-1, 4, 4, 2)).movedim(-4, -3).movedim(-1, -2).flatten(-4).unflatten(-1, (-1, 2))
    return w[..., 0] | (w[..., 1] << 4)


def k_codes(row):
    w = torch.stack([row & 15, row >> 4], -1).flatten(-2).unflatten(-1, (4, -1, 2, 4))
    return w.movedim(-1, -2).movedim(-4, -3).flatten(-4)


def exchanged(row, at):
    """Rows of 64 bytes: the second pair of every four rows of a block has its 32-byte halves exchanged."""
    return row if row.shape[-1] != 64 else torch.where((at >> 1 & 1).bool()[..., None], row.roll(32, -1), row)


def v_bytes(code, at):
    """Codes [..., dim] of a value as its row of bytes, `at` its row in the block."""
    w = code.unflatten(-1, (-1, 2, 8, 4)).movedim(-2, -4).flatten(-4).unflatten(-1, (-1, 2))
    return exchanged(w[..., 0] | (w[..., 1] << 4), at)


def v_codes(row, at):
    w = torch.stack([exchanged(row, at) & 15, exchanged(row, at) >> 4], -1).flatten(-2).unflatten(-1, (8, -1, 2, 4))
    return w.movedim(-4, -2).flatten(-4)


def pack(k, v, kp, vp):
    """Codes [..., page, dim] (uint8 values 0-15) and parameters [..., page, groups, 2] as the bytes of their records."""
    page = k.shape[-2]
    block = min(page, 32)
    rows = v_row(torch.arange(block, device=k.device))
    kb, vc = k_bytes(k).unflatten(-2, (-1, block)), v.unflatten(-2, (-1, block))
    vb = torch.empty_like(kb)
    vb[..., rows, :] = v_bytes(vc, rows)
    par = [x.contiguous().view(torch.uint8).flatten(-2).unflatten(-2, (-1, block)) for x in (kp, vp)]
    return torch.cat([x.flatten(-2) for x in (kb, vb, *par)], -1).flatten(-2)


def values(code, par):
    """scale * code + minimum, fp32, of codes [..., dim] and parameters [..., groups, 2]."""
    x = code.unflatten(-1, (par.shape[-2], -1)).float()
    return (x * par[..., 0:1].float() + par[..., 1:2].float()).flatten(-2)


def unpack(records, page, dim, group, dtype):
    """The dequantised K and V, fp32 [..., page, dim], of records [..., bytes]."""
    block = min(page, 32)
    rows = v_row(torch.arange(block, device=records.device))
    r = records.unflatten(-1, (page // block, -1))
    half, some = block * dim // 2, block * 4 * (dim // group)
    kb, vb, kp, vp = torch.split(r, [half, half, some, some], -1)
    kb, vb = kb.unflatten(-1, (block, -1)), vb.unflatten(-1, (block, -1))[..., rows, :]
    kp, vp = (x.contiguous().view(dtype).unflatten(-1, (block, -1, 2)) for x in (kp, vp))
    return values(k_codes(kb), kp).flatten(-3, -2), values(v_codes(vb, rows), vp).flatten(-3, -2)


def quantise(x, group):
    """Codes (uint8) and parameters (scale, minimum) of x [..., dim] in groups along the last axis."""
    g = x.reshape(*x.shape[:-1], -1, group).float()
    mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((mx * 0.5 - mn * 0.5) / 7.5).to(x.dtype)
    step = scale.float()
    code = torch.where(step > 0, torch.round((g - mn) / step), torch.zeros_like(g)).clamp(0, 15)
    return code.to(torch.uint8).view(x.shape), torch.stack([scale, mn.to(x.dtype)], -1).squeeze(-2)


# --------------------------------------------------------------------------------------------------------------------
# Page bookkeeping on the host, for the state that a program starts from
# --------------------------------------------------------------------------------------------------------------------
def spare(case):
    return -(-case["longest"] // case["page"]) + case["slots"]


def page_state(case):
    """Lengths, table rows, counts of a cache that requests of interleaved arrival have filled, and its table's width."""
    lens, ps = lengths(case, case["slots"], case["longest"]), case["page"]
    width = -(-case["longest"] // ps) + 2
    table, used = [[] for _ in lens], 0
    for depth in range(width):
        for s, n in enumerate(lens):
            if depth * ps < n:
                table[s].append(used)
                used += 1
    extra = used if case["act"] == "copy" else 0
    return lens, table, [1] * used + [0] * (extra + spare(case)), width


def page_moves(case, lens, table):
    ps, half = case["page"], case["slots"] // 2
    if case["act"] == "fork":
        return sum(1 for s in range(half) if lens[2 * s] % ps)
    if case["act"] == "copy":
        return sum(len(table[2 * s]) for s in range(half))
    live = [p for s, row in enumerate(table) if not (s % 2 and s // 2 < half) for p in row]
    return sum(1 for p in live if p >= len(live))


# --------------------------------------------------------------------------------------------------------------------
# States
# --------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    return {"prompt": prepare_prompt, "decode": prepare_decode, "store": prepare_store, "pages": prepare_pages}[case["op"]](
        case, torch.Generator("cuda").manual_seed(seed))


def normal(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare_prompt(case, gen):
    dt, d, hq, hkv = DTYPES[case["dtype"]], case["dim"], case["hq"], case["hkv"]
    ql, kl = prompt_lengths(case)
    s = {"case": case, "cuq": whole(starts(ql)), "cuk": whole(starts(kl)), "longest": (max(ql), max(kl)),
         "o": torch.zeros(sum(ql), hq, d, dtype=dt, device="cuda")}
    if case["prefix"]:
        s["q"] = normal(gen, sum(ql), hq, d, dtype=dt)
        s["k"] = normal(gen, sum(kl), hkv, d, dtype=dt)
        s["v"] = normal(gen, sum(kl), hkv, d, dtype=dt)
    else:
        s["qkv"] = normal(gen, sum(ql), hq + 2 * hkv, d, dtype=dt)
    return s


def prepare_cache(case, gen, lens, width, fill):
    """A pool whose pages hold a quantised normal history, a table of shuffled pages and the lengths."""
    dt, d, hkv, ps, g = DTYPES[case["dtype"]], case["dim"], case["hkv"], case["page"], case["group"]
    counts = [-(-n // ps) for n in lens]
    total = sum(counts) + 3
    pool = torch.zeros(total, page_bytes(case), dtype=torch.uint8, device="cuda")
    if fill:
        step = max(1, (1 << 25) // (hkv * ps * d))
        # A key channel has its own spread, as rotated keys do.
        spread = 0.5 + torch.rand(d, generator=gen, device="cuda") * 1.5
        for lo in range(0, total, step):
            n = min(step, total - lo)
            k = (torch.randn(n, hkv, ps, d, generator=gen, device="cuda") * spread).to(dt)
            v = normal(gen, n, hkv, ps, d, dtype=dt)
            (kc, kp), (vc, vp) = quantise(k, g), quantise(v, g)
            pool[lo:lo + n] = pack(kc, vc, kp, vp).flatten(1)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return {"pool": pool, "table": table, "lens": whole(lens), "pages": total}


def prepare_decode(case, gen):
    dt, d, hq = DTYPES[case["dtype"]], case["dim"], case["hq"]
    lens = lengths(case, case["slots"], case["longest"])
    s = prepare_cache(case, gen, lens, -(-case["longest"] // case["page"]), True)
    s.update(case=case, q=normal(gen, case["slots"], hq, d, dtype=dt), longest=case["longest"],
             o=torch.zeros(case["slots"], hq, d, dtype=dt, device="cuda"))
    return s


def prepare_store(case, gen):
    dt, d, hkv = DTYPES[case["dtype"]], case["dim"], case["hkv"]
    new = lengths(case, case["slots"], case["longest"])
    old = [n - 1 for n in lengths(case, case["slots"], case["context"] + 1, 1)]
    lens = [a + b for a, b in zip(new, old)]
    s = prepare_cache(case, gen, lens, -(-max(lens) // case["page"]), False)
    total = sum(new)
    s.update(case=case, cu=whole(starts(new)), k=normal(gen, total, hkv, d, dtype=dt), v=normal(gen, total, hkv, d, dtype=dt),
             k_back=torch.zeros(total, hkv, d, dtype=dt, device="cuda"), v_back=torch.zeros(total, hkv, d, dtype=dt, device="cuda"))
    return s


def prepare_pages(case, gen):
    lens, rows, refs, width = page_state(case)
    table = whole([r + [-1] * (width - len(r)) for r in rows])
    pool = torch.randint(0, 256, (case["layers"], len(refs), page_bytes(case)), generator=gen, device="cuda", dtype=torch.uint8)
    half = case["slots"] // 2
    odd = whole([2 * s + 1 for s in range(half)])
    even = whole([2 * s for s in range(half)])
    fresh = lengths(case, half, case["longest"], 2)
    # New requests that fit the pages which the leaving ones free.
    fresh = [min(n, lens[2 * s + 1]) for s, n in enumerate(fresh)]
    back = [min(n, lens[2 * s]) for s, n in enumerate(lengths(case, half, case["longest"], 3))]
    return {"case": case, "table": table, "lens": whole(lens), "refs": whole(refs), "pool": pool, "src": even, "dst": odd,
            "leave0": odd, "leave1": even, "fresh0": whole(fresh), "fresh1": whole(back), "turn": 0, "pages": len(refs)}


# --------------------------------------------------------------------------------------------------------------------
# Runs
# --------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"prompt": own_prompt, "decode": own_decode, "store": own_store, "pages": own_pages}[op](state)
    return {"prompt": plain_prompt, "decode": plain_decode, "store": plain_store, "pages": plain_pages}[op](state)


def attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v of q [b, h, per, i, d], k and v [b, h, j, d]; `seen` [b, i, j]: which keys a row sees."""
    s = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(scale)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    return torch.matmul(p, v[:, :, None]) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def plain_prompt(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["dim"]
    if "qkv" in s:
        q, k, v = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:]
    else:
        q, k, v = s["q"], s["k"], s["v"]
    ql, kl = s["cuq"][1:] - s["cuq"][:-1], s["cuk"][1:] - s["cuk"][:-1]
    i, j = torch.arange(s["longest"][0], device=q.device), torch.arange(s["longest"][1], device=q.device)
    rows = (s["cuq"][:-1, None] + i).clamp_max(q.shape[0] - 1)
    keys = (s["cuk"][:-1, None] + j).clamp_max(k.shape[0] - 1)
    q = q[rows].float().permute(0, 2, 1, 3).unflatten(1, (hkv, hq // hkv))
    k, v = k[keys].float().transpose(1, 2), v[keys].float().transpose(1, 2)
    seen = (j < kl[:, None])[:, None] & (j <= (i + (kl - ql)[:, None])[:, :, None])
    o = attend(q, k, v, seen, 1 / math.sqrt(d)).flatten(1, 2).transpose(1, 2)
    t = torch.arange(s["o"].shape[0], device=q.device, dtype=torch.int32)
    b = torch.searchsorted(s["cuq"], t, right=True) - 1
    return o[b, t - s["cuq"][b]].to(s["o"].dtype)


def plain_decode(s):
    c = s["case"]
    hq, hkv, d, ps = c["hq"], c["hkv"], c["dim"], c["page"]
    records = s["pool"].view(s["pages"], hkv, -1)[s["table"].clamp_min(0).long()]
    k, v = unpack(records, ps, d, c["group"], s["q"].dtype)
    k, v = k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)
    seen = (torch.arange(k.shape[2], device=k.device) < s["lens"][:, None])[:, None]
    v = v.masked_fill_(~seen[:, :, :, None], 0)
    q = s["q"].float().view(c["slots"], hkv, hq // hkv, 1, d)
    # The rows of one cached head meet its keys in one product.
    o = attend(q.transpose(2, 3), k, v, seen.expand(-1, hq // hkv, -1), 1 / math.sqrt(d))
    return o.reshape(c["slots"], hq, d).to(s["o"].dtype)


def places(s):
    """Pool page and place in it of every new token: token i of a slot's n ends at the slot's length."""
    t = torch.arange(s["k"].shape[0], device=s["k"].device, dtype=torch.int32)
    b = torch.searchsorted(s["cu"], t, right=True) - 1
    at = s["lens"][b] - s["cu"][b + 1] + t
    return s["table"][b, at // s["case"]["page"]].long(), at % s["case"]["page"]


def plain_store(s):
    c = s["case"]
    d, hkv, dt = c["dim"], c["hkv"], s["k"].dtype
    page, at = places(s)
    block, ng = min(c["page"], 32), d // c["group"]
    r = at % block
    vr = v_row(r)
    (kc, kp), (vc, vp) = quantise(s["k"], c["group"]), quantise(s["v"], c["group"])
    token = torch.cat([k_bytes(kc), v_bytes(vc, vr[:, None]), kp.view(torch.uint8).flatten(-2), vp.view(torch.uint8).flatten(-2)], -1)
    i, j = torch.arange(d // 2, device=page.device), torch.arange(4 * ng, device=page.device)
    r, vr = r[:, None], vr[:, None]
    place = torch.cat([r * (d // 2) + i, (block + vr) * (d // 2) + i, block * d + r * 4 * ng + j,
                       block * d + (block + r) * 4 * ng + j], -1)
    place = (place + (at // block)[:, None] * (block * (d + 8 * ng)))[:, None]
    pool = s["pool"].view(s["pages"], hkv, -1)
    h = torch.arange(hkv, device=page.device)[None, :, None]
    pool[page[:, None, None], h, place] = token
    token = pool[page[:, None, None], h, place]
    kb, vb, kp, vp = torch.split(token, [d // 2, d // 2, 4 * ng, 4 * ng], -1)
    kp, vp = (x.contiguous().view(dt).unflatten(-1, (-1, 2)) for x in (kp, vp))
    return values(k_codes(kb), kp).to(dt), values(v_codes(vb, vr), vp).to(dt)


def plain_free(s, ids):
    width, ps = s["table"].shape[1], s["case"]["page"]
    ids = ids.long()
    held = torch.arange(width, device=ids.device) * ps < s["lens"][ids][:, None]
    rows = s["table"][ids]
    s["refs"].index_add_(0, rows.clamp_min(0).flatten().long(), -held.flatten().int())
    s["table"][ids] = torch.where(held, -1, rows)
    s["lens"][ids] = 0


def free_order(s):
    return torch.sort((s["refs"] > 0).int(), stable=True)[1].int()


def plain_grow(s, ids, add):
    ps, width = s["case"]["page"], s["table"].shape[1]
    ids = ids.long()
    old = s["lens"][ids]
    have, want = (old + ps - 1) // ps, (old + add + ps - 1) // ps
    base = torch.cumsum(want - have, 0).int() - (want - have)
    col = torch.arange(width, device=ids.device)
    new = (col >= have[:, None]) & (col < want[:, None])
    order = free_order(s)
    taken = order[(base[:, None] + col - have[:, None]).clamp(0, order.shape[0] - 1).long()]
    s["table"][ids] = torch.where(new, taken, s["table"][ids])
    s["refs"].index_add_(0, torch.where(new, taken, 0).flatten().long(), new.flatten().int())
    s["lens"][ids] = old + add


def plain_fork(s, src, dst, deep):
    ps, width = s["case"]["page"], s["table"].shape[1]
    src, dst = src.long(), dst.long()
    n = s["lens"][src]
    held = (n + ps - 1) // ps
    share = torch.zeros_like(n) if deep else n // ps
    base = torch.cumsum(held - share, 0).int() - (held - share)
    col = torch.arange(width, device=src.device)
    rows = s["table"][src]
    kept, new = col < share[:, None], (col >= share[:, None]) & (col < held[:, None])
    order = free_order(s)
    taken = order[(base[:, None] + col - share[:, None]).clamp(0, order.shape[0] - 1).long()]
    child = torch.where(kept, rows, torch.where(new, taken, s["table"][dst]))
    s["table"][dst] = child
    counted = kept | new
    s["refs"].index_add_(0, torch.where(counted, child, 0).flatten().long(), counted.flatten().int())
    s["lens"][dst] = n
    if deep:
        where = new
        a, b = rows[where].long(), taken[where].long()
    else:  # at most one new page a fork: its last
        last = share.long()[:, None].clamp_max(width - 1)
        part = (held > share)[:, None]
        a = torch.gather(rows, 1, last)[part].long()
        b = torch.gather(taken, 1, last)[part].long()
    s["pool"][:, b] = s["pool"][:, a]


def plain_compact(s):
    live = s["refs"] > 0
    count = live.sum()
    page = torch.arange(live.shape[0], device=live.device)
    hole, mover = page[(page < count) & ~live], page[(page >= count) & live]
    to = page.clone()
    to[mover] = hole
    s["pool"][:, hole] = s["pool"][:, mover]
    s["refs"][hole] = s["refs"][mover]
    s["refs"][mover] = 0
    ps, width = s["case"]["page"], s["table"].shape[1]
    held = torch.arange(width, device=live.device) * ps < s["lens"][:, None]
    s["table"].copy_(torch.where(held, to[s["table"].clamp_min(0).long()].int(), s["table"]))


def plain_pages(s):
    if s["case"]["act"] == "turnover":
        leave, fresh = s["leave%d" % s["turn"]], s["fresh%d" % s["turn"]]
        s["turn"] ^= 1
        plain_free(s, leave)
        plain_compact(s)
        plain_grow(s, leave, fresh)
    else:
        plain_free(s, s["dst"])
        plain_fork(s, s["src"], s["dst"], s["case"]["act"] == "copy")
    return s["table"], s["lens"], s["refs"], s["pool"]


# --------------------------------------------------------------------------------------------------------------------
# The framework's operators
# --------------------------------------------------------------------------------------------------------------------
def builders():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorchsim-triton-backend_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from pytorchsim_triton_compiler.codegen import build
    return build


def graph(s, key, steps):
    """Runs the launch graph of `steps` [(descriptor, names of its buffers)], built once over a state's buffers."""
    if key not in s:
        builders()
        from pytorchsim_triton_compiler.codegen import descriptors as D
        from pytorchsim_triton_compiler.runtime.graph import Graph
        g = Graph("cuda:%d" % torch.cuda.current_device())
        for i, (desc, names) in enumerate(steps()):
            for n in names:
                g.bind(n, s[n])
            g.add("step%d" % i, D.to_bytes(desc), names)
        s[key] = g
    s[key].run()


def own_prompt(s):
    def steps():
        c, B = s["case"], builders()
        if "qkv" in s:
            return [(B.attention_packed(s["o"].shape[0], c["seqs"], c["hq"], c["hkv"], c["dim"], dtype=c["dtype"], fused=True),
                     ["qkv", "cuq", "o"])]
        return [(B.attention_packed(s["o"].shape[0], c["seqs"], c["hq"], c["hkv"], c["dim"], dtype=c["dtype"],
                                    k_tokens=s["k"].shape[0]), ["q", "k", "v", "cuq", "cuk", "o"])]
    graph(s, "graph", steps)
    return s["o"]


def cache_of(s):
    c = s["case"]
    return builders().kv4_cache(slots=c["slots"], max_pages=s["table"].shape[1], pages=s["pages"], hkv=c["hkv"], dim=c["dim"],
                                page_size=c["page"], group=c["group"], layers=c.get("layers", 1), dtype=c.get("dtype", "bfloat16"))


def own_decode(s):
    graph(s, "graph", lambda: [(builders().attention_kv4(cache_of(s), s["case"]["hq"]), ["q", "lens", "table", "pool", "o"])])
    return s["o"]


def own_store(s):
    n = s["k"].shape[0]
    graph(s, "graph", lambda: [(builders().kv4_store(cache_of(s), n), ["k", "v", "cu", "lens", "table", "pool"]),
                               (builders().kv4_load(cache_of(s), n), ["cu", "lens", "table", "pool", "k_back", "v_back"])])
    return s["k_back"], s["v_back"]


def own_pages(s):
    books, n = ["table", "lens", "refs"], s["case"]["slots"] // 2
    if s["case"]["act"] == "turnover":
        turn = s["turn"]
        s["turn"] ^= 1
        graph(s, "graph%d" % turn, lambda: [
            (builders().pages_free(cache_of(s), n), ["leave%d" % turn] + books),
            (builders().pages_compact(cache_of(s)), books + ["pool"]),
            (builders().pages_grow(cache_of(s), n), ["leave%d" % turn, "fresh%d" % turn] + books)])
    else:
        graph(s, "graph", lambda: [
            (builders().pages_free(cache_of(s), n), ["dst"] + books),
            (builders().pages_fork(cache_of(s), n, deep=s["case"]["act"] == "copy"), ["src", "dst"] + books + ["pool"])])
    return s["table"], s["lens"], s["refs"], s["pool"]


# --------------------------------------------------------------------------------------------------------------------
# In 64 bits, from the definitions
# --------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    return {"prompt": exact_prompt, "decode": exact_decode, "store": exact_store}[case["op"]](case, s)


def exact_prompt(case, s):
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    if "qkv" in s:
        q, k, v = torch.split(s["qkv"], [hq, hkv, hkv], dim=1)
    else:
        q, k, v = s["q"], s["k"], s["v"]
    ql, kl = prompt_lengths(case)
    cq, ck = starts(ql), starts(kl)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        keys = torch.arange(kl[b], device="cuda")
        place = torch.arange(ql[b], device="cuda") + (kl[b] - ql[b])
        hidden = keys[None, :] > place[:, None]
        for h in range(hq):
            kd = k[ck[b]:ck[b + 1], h * hkv // hq].double()
            vd = v[ck[b]:ck[b + 1], h * hkv // hq].double()
            z = (q[cq[b]:cq[b + 1], h].double() @ kd.T) / math.sqrt(d)
            z[hidden] = -math.inf
            out[cq[b]:cq[b + 1], h] = torch.softmax(z, dim=1) @ vd
    return out


def exact_rows(record, token, dim, group, page, dtype, which):
    """The values of K (which 0) or V (1) at `token` of a record, [dim] in 64 bits, code by code from the format."""
    block = min(page, 32)
    size = block * (dim + 8 * (dim // group))
    base = (token // block) * size
    t = (token % block)[..., None]
    d = torch.arange(dim, device=record.device)
    if which == 0:
        inside = d % 32
        word = (inside // 8) * (dim // 32) + d // 32
        nibble = (inside % 8) // 2 + 4 * (inside % 2)
        row = t
    else:
        row = (t // 8) * 8 + (t % 2) * 4 + (t % 8) // 2
        lane = (d % 32) // 4
        if dim == 128:
            lane = lane ^ (4 * ((row // 2) % 2))
        word = lane * (dim // 64) + d // 64
        nibble = d % 4 + 4 * ((d % 64) // 32)
    at = base[..., None] + which * (block * dim // 2) + row * (dim // 2) + word * 4 + nibble // 2
    code = (torch.gather(record, -1, at).int() >> (4 * (nibble % 2))) & 15
    par = base[..., None] + block * dim + which * block * 4 * (dim // group) + t * 4 * (dim // group)
    at = par + torch.arange(4 * (dim // group), device=record.device)
    p = torch.gather(record, -1, at).contiguous().view(dtype).double().unflatten(-1, (dim // group, 2))
    return code.double() * p[..., 0].repeat_interleave(group, -1) + p[..., 1].repeat_interleave(group, -1)


def exact_decode(case, s):
    hq, hkv, d, ps = case["hq"], case["hkv"], case["dim"], case["page"]
    lens = lengths(case, case["slots"], case["longest"])
    pool = s["pool"].view(s["pages"], hkv, -1)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        page = s["table"][b, t // ps].long()
        for h in range(hkv):
            kv = []
            for which in (0, 1):
                parts = []
                for lo in range(0, n, 16384):
                    records = pool[s["table"][b, lo // ps:-(-min(n, lo + 16384) // ps)].long(), h]
                    inside = torch.arange(ps, device="cuda").expand(records.shape[0], ps)
                    wide = records[:, None].expand(-1, ps, -1)
                    parts.append(exact_rows(wide, inside, d, case["group"], ps, s["q"].dtype, which).flatten(0, 1))
                kv.append(torch.cat(parts)[:n])
            rows = slice(h * hq // hkv, (h + 1) * hq // hkv)
            z = (s["q"][b, rows].double() @ kv[0].T) / math.sqrt(d)
            out[b, rows] = torch.softmax(z, dim=1) @ kv[1]
    return out


def exact_store(case, s):
    def back(x):
        g = x.double().unflatten(-1, (-1, case["group"]))
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        step = ((high - low) / 15).to(x.dtype).double()
        code = torch.round((g - low) / torch.where(step > 0, step, 1)).clamp(0, 15)
        return (code * step + low).flatten(-2)
    return back(s["k"]), back(s["v"])
