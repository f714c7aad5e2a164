"""CPU oracle of the serving operators in 64 bits -- TEST INFRASTRUCTURE ONLY: packed prompt attention, the 4-bit paged
cache (quantisation, record format, one-token attention) and the page bookkeeping.  They have no program in the
reference; each function states the operator's definition (include/ptsim_b200.h) value by value or slot by slot."""
import math

import torch


def attention_packed(q, k, v, cuq, cuk, scale, o):
    """q [Tq, hq, D], k, v [Tk, hkv, D]; query i of a sequence sees keys j <= i + kl - ql; rows outside every sequence
    keep `o`'s values.  Returns float64."""
    out = o.double().clone()
    per = q.shape[1] // k.shape[1]
    for s in range(len(cuq) - 1):
        ql, kl = cuq[s + 1] - cuq[s], cuk[s + 1] - cuk[s]
        for i in range(ql):
            n = min(kl, i + kl - ql + 1)
            row = cuq[s] + i
            if n <= 0:
                out[row] = 0
                continue
            keys = k[cuk[s]:cuk[s] + n].double().repeat_interleave(per, 1)
            vals = v[cuk[s]:cuk[s] + n].double().repeat_interleave(per, 1)
            z = torch.einsum("hd,nhd->hn", q[row].double(), keys) * scale
            out[row] = torch.einsum("hn,nhd->hd", torch.softmax(z, 1), vals)
    return out


def quantise(x, group):
    """(codes int64 [..., D], scale, minimum [..., D / group]) of x, in the arithmetic of its definition: fp32 quotients of halves."""
    g = x.unflatten(-1, (-1, group)).float()
    mn, mx = g.amin(-1), g.amax(-1)
    scale = ((mx * 0.5 - mn * 0.5) / 7.5).to(x.dtype)
    bad = ~torch.isfinite(mx * 0.5 - mn * 0.5)
    half = scale.float()[..., None] * 0.5          # halves throughout: exact, and the largest range does not overflow
    code = torch.where(half > 0, torch.round((g * 0.5 - mn[..., None] * 0.5) / half), 0.0).clamp(0, 15)
    code = torch.where(bad[..., None], 0.0, code)
    nan = float("nan")
    return (code.to(torch.int64).flatten(-2), torch.where(bad, nan, scale.float()).to(x.dtype),
            torch.where(bad, nan, mn).to(x.dtype))


def dequantised(x, group):
    """What the cache stands for after x went in, float64."""
    code, scale, mn = quantise(x, group)
    c = code.unflatten(-1, (-1, group)).double()
    return (c * scale.double()[..., None] + mn.double()[..., None]).flatten(-2)


def token_bytes(at, page_size, dim, group):
    """Byte of every value's code (and which nibble) and of every group's (scale, minimum) of K and V of the token at place
    `at` of a page, within the record of one KV head."""
    b = min(page_size, 32)
    ng = dim // group
    base, t = at // b * (b * (dim + 8 * ng)), at % b
    r = (t & ~7) | ((t & 1) << 2) | ((t >> 1) & 3)
    k, v = [], []
    for d in range(dim):
        word, nib = (d % 32 // 8) * (dim // 32) + d // 32, (d % 8) // 2 + 4 * (d % 2)
        k.append((base + t * (dim // 2) + word * 4 + nib // 2, nib % 2))
        c = d % 32 // 4
        if dim == 128 and r & 2:
            c ^= 4
        word, nib = c * (dim // 64) + d // 64, d % 4 + 4 * (d % 64 // 32)
        v.append((base + b * (dim // 2) + r * (dim // 2) + word * 4 + nib // 2, nib % 2))
    par = base + b * dim
    kp = [par + (t * ng + i) * 4 for i in range(ng)]
    vp = [par + (b * ng + t * ng + i) * 4 for i in range(ng)]
    return k, v, kp, vp


class Cache:
    """A 4-bit paged cache held as dense values, and its pool's bytes."""

    def __init__(self, shape, pool, table, lens):
        self.s, self.table, self.lens = shape, table, lens
        self.pool = pool.view(shape.layers, shape.pages, shape.hkv, -1).clone()
        self.dtype = getattr(torch, shape.dtype)
        self.where = [token_bytes(t, shape.page_size, shape.dim, shape.group) for t in range(shape.page_size)]

    def write(self, slot, pos, head, k, v, layer=0):
        rec = self.pool[layer, self.table[slot][pos // self.s.page_size], head]
        for x, places, params in zip((k, v), self.where[pos % self.s.page_size][:2], self.where[pos % self.s.page_size][2:]):
            code, scale, mn = quantise(x, self.s.group)
            for c, (byte, hi) in zip(code.tolist(), places):
                rec[byte] = (int(rec[byte]) & (0x0f if hi else 0xf0)) | (c << (4 if hi else 0))
            for i, at in enumerate(params):
                rec[at:at + 4] = torch.stack([scale[i], mn[i]]).view(torch.uint8)

    def read(self, slot, pos, head, layer=0):
        rec = self.pool[layer, self.table[slot][pos // self.s.page_size], head]
        out = []
        w = self.where[pos % self.s.page_size]
        for places, params in ((w[0], w[2]), (w[1], w[3])):
            code = torch.tensor([(int(rec[byte]) >> (4 if hi else 0)) & 15 for byte, hi in places], dtype=torch.float64)
            par = torch.stack([rec[at:at + 4].clone().view(self.dtype).double() for at in params])
            out.append((code.unflatten(0, (-1, self.s.group)) * par[:, :1] + par[:, 1:]).flatten())
        return out

    def attend(self, q, scale, layer=0):
        out = torch.zeros(q.shape, dtype=torch.float64)
        per = q.shape[1] // self.s.hkv
        for slot, n in enumerate(self.lens):
            for h in range(self.s.hkv if n else 0):
                kv = [self.read(slot, p, h, layer) for p in range(n)]
                k, v = (torch.stack([x[i] for x in kv]) for i in (0, 1))
                z = q[slot, h * per:(h + 1) * per].double() @ k.T * scale
                out[slot, h * per:(h + 1) * per] = torch.softmax(z, 1) @ v
        return out


class Pages:
    """The page bookkeeping slot by slot: lists of pages, counts, and a pool of [layers, pages, bytes]."""

    def __init__(self, table, lens, refs, pool, page_size):
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)
        self.pool, self.ps = pool.clone(), page_size

    def held(self, n):
        return -(-n // self.ps)

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def grow(self, ids, add):
        for s, n in zip(ids, add):
            for k in range(self.held(self.lens[s]), self.held(self.lens[s] + n)):
                self.table[s][k] = self.take()
            self.lens[s] += n

    def fork(self, src, dst, deep=False):
        # The pages are taken in list order first: shared pages are counted after them, and are in use anyway.
        for a, b in zip(src, dst):
            n = self.lens[a]
            full = 0 if deep else n // self.ps
            for k in range(self.held(n)):
                if k < full:
                    self.table[b][k] = self.table[a][k]
                    self.refs[self.table[a][k]] += 1
                else:
                    self.table[b][k] = self.take()
                    self.pool[:, self.table[b][k]] = self.pool[:, self.table[a][k]]
            self.lens[b] = n

    def free(self, ids):
        for s in ids:
            for k in range(self.held(self.lens[s])):
                self.refs[self.table[s][k]] -= 1
                self.table[s][k] = -1
            self.lens[s] = 0

    def compact(self):
        used = [p for p, r in enumerate(self.refs) if r > 0]
        holes = [p for p in range(len(used)) if self.refs[p] <= 0]
        to = dict(zip([p for p in used if p >= len(used)], holes))
        for a, b in to.items():
            self.pool[:, b] = self.pool[:, a]
            self.refs[a], self.refs[b] = 0, self.refs[a]
        for s, n in enumerate(self.lens):
            for k in range(self.held(n)):
                self.table[s][k] = to.get(self.table[s][k], self.table[s][k])
