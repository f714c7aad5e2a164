"""The serving operators on the B200 against their definitions in 64 bits (oracle/serving.py and dense float64 products):
packed prompt attention, the 4-bit paged cache, the page bookkeeping, and a serving loop of all of them.

Tolerances, from the roundings that the kernels make (eps: the 16-bit type's; half a step is eps / 2):
  - attention: each weight p_j is rounded to the type before it multiplies v_j, an error of at most eps / 2 of it, so a result
    moves by at most eps / 2 times A = sum_j softmax_j |v_j|; the result itself is rounded, eps / 2 |o|.  The fp32 work (products
    of 128 terms, the exponential, the sums) adds at most 2^-13 A: scores here are at most 2^4 with an error below
    2^-20 of the sum of their absolute products (2^5 at most), 2^-15 twice, and the sums 2^-17.  fp16 adds half its
    smallest step, 2^-25, where results are that small;
  - over the cache: the rounded weight is p_j a_j (a: the V scale) and multiplies |code - 8| <= 8: eps / 2 * 8 sum_j softmax_j a_j in
    the place of eps / 2 A;
  - store: the record's bytes are those of the definition; load: one fp32 fma rounded to the type, eps / 2 of the value plus
    2^-24 of scale * 15 + |minimum| for the fma;
  - page bookkeeping: equal."""
import math

import pytest
import torch

from oracle import serving as S
from pytorchsim_triton_compiler.codegen import build as B
from pytorchsim_triton_compiler.codegen import descriptors as D
from pytorchsim_triton_compiler.runtime import cuda as RC
from pytorchsim_triton_compiler.runtime import native
from pytorchsim_triton_compiler.runtime.graph import Graph

pytestmark = pytest.mark.gpu

DT = {"bfloat16": torch.bfloat16, "float16": torch.float16}
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def launch(desc, tensors, **kw):
    return RC.launch_tensors(D.to_bytes(desc), tensors, **kw)


def failed(desc, tensors):
    with pytest.raises(native.ExecutorError) as e:
        launch(desc, tensors)
    return e.value.code


# --------------------------------------------------------------------------------------------------------------------
# Packed prompt attention
# --------------------------------------------------------------------------------------------------------------------
def dense(q, k, v, ql, kl, q0, k0, scale):
    """(o, A) in float64 on the GPU: per sequence, per head."""
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    per = q.shape[1] // k.shape[1]
    for s in range(len(ql)):
        for h in range(q.shape[1]):
            qq, kk, vv = (x[a:a + n, i].double() for x, a, n, i in ((q, q0[s], ql[s], h), (k, k0[s], kl[s], h // per), (v, k0[s], kl[s], h // per)))
            place = torch.arange(ql[s], device=q.device)[:, None] + kl[s] - ql[s]
            z = (qq @ kk.T * scale).masked_fill(torch.arange(kl[s], device=q.device)[None] > place, -math.inf)
            p = torch.softmax(z, 1).nan_to_num(0.0) if kl[s] else z
            out[q0[s]:q0[s] + ql[s], h], mag[q0[s]:q0[s] + ql[s], h] = p @ vv, p @ vv.abs()
    return out, mag


def near(got, want, mag, dtype, what=""):
    half = torch.finfo(dtype).eps / 2
    bound = half * (mag + want.abs()) + 2.0 ** -13 * mag + SMALLEST[dtype] + 1e-300
    off = ((got.double() - want).abs() / bound)
    assert bool((off <= 1).all()), f"{what}: {float(off.max()):.2f} of the bound at {divmod(int(off.argmax()), got.shape[-1])}"


def packed_case(ql, kl, hq, hkv, dim, dtype, seed, gap=0, tail=0):
    """Random rows; `gap` rows before the first sequence and `tail` after the last are in none."""
    dt, g = DT[dtype], gen(seed)
    q0, k0 = starts(ql, gap), starts(kl, gap)
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dt).cuda() for n, h in
               ((q0[-1] + tail, hq), (k0[-1] + tail, hkv), (k0[-1] + tail, hkv)))
    return q, k, v, q0, k0


LENS = [[1], [2, 1, 3], [128], [129], [127, 1, 256], [257, 0, 255, 0, 0, 64], [0, 0, 300], [640, 33, 1, 511]]


@pytest.mark.parametrize("dim,dtype,hq,hkv", [(128, "bfloat16", 4, 2), (64, "float16", 3, 1), (128, "float16", 2, 2), (64, "bfloat16", 8, 1)])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_packed_attention(lens, dim, dtype, hq, hkv):
    q, k, v, q0, k0 = packed_case(lens, lens, hq, hkv, dim, dtype, sum(lens) + dim)
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(q0[-1], len(lens), hq, hkv, dim, dtype=dtype), [q, k, v, ints(q0), o])
    near(o, *dense(q, k, v, lens, lens, q0, k0, 1 / math.sqrt(dim)), DT[dtype])


@pytest.mark.parametrize("dim,dtype", [(128, "bfloat16"), (64, "float16")])
@pytest.mark.parametrize("ql,kl", [([1], [1000]), ([5, 200], [5, 333]), ([300], [100]), ([129, 2, 7], [0, 1, 700]), ([256, 256], [511, 383]),
                                   ([400], [1]), ([257], [256])], ids=str)
def test_packed_attention_with_cached_prefixes(ql, kl, dim, dtype):
    """More keys than queries (a chunk behind a prefix), fewer (rows that see nothing give zeros), none."""
    q, k, v, q0, k0 = packed_case(ql, kl, 4, 2, dim, dtype, sum(kl))
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(q0[-1], len(ql), 4, 2, dim, dtype=dtype, k_tokens=k0[-1]), [q, k, v, ints(q0), ints(k0), o])
    want, mag = dense(q, k, v, ql, kl, q0, k0, 1 / math.sqrt(dim))
    near(o, want, mag, DT[dtype])
    for s in range(len(ql)):
        hidden = max(0, ql[s] - kl[s])
        assert not o[q0[s]:q0[s] + hidden].any()


# Averages of 768 keys (dim 128) and 4096 (dim 64) and more run two query tiles a CTA.
@pytest.mark.parametrize("ql,kl,dim,dtype", [
    ([1025, 3, 1400], [1025, 3, 1400], 128, "bfloat16"), ([257, 1, 128, 640], [2000, 900, 128, 641], 128, "float16"),
    ([300, 129, 0, 5], [5000, 4300, 9000, 6], 64, "bfloat16"), ([1500], [800], 128, "bfloat16"), ([513, 256], [4096, 4351], 64, "float16")], ids=str)
def test_packed_attention_of_long_sequences(ql, kl, dim, dtype):
    q, k, v, q0, k0 = packed_case(ql, kl, 3, 1, dim, dtype, sum(kl))
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(q0[-1], len(ql), 3, 1, dim, dtype=dtype, k_tokens=k0[-1]), [q, k, v, ints(q0), ints(k0), o])
    near(o, *dense(q, k, v, ql, kl, q0, k0, 1 / math.sqrt(dim)), DT[dtype])


@pytest.mark.parametrize("dim,dtype,more,keys", [(128, "bfloat16", 700, 800), (128, "float16", 1152, 1024), (64, "bfloat16", 700, 4200)])
def test_rows_without_keys_beside_a_tile_with_keys_are_zeros(dim, dtype, more, keys):
    """`more` queries than keys: the first item with a key has none in its first tile.  The zeros of those rows take the place of Q
    in shared memory, so Q of such a tile must not be on its way there."""
    ql, kl = [keys + more + i % 3 for i in range(12)], [keys] * 12
    assert all(128 <= (a - b) % 256 < 256 for a, b in zip(ql, kl))
    q, k, v, q0, k0 = packed_case(ql, kl, 4, 1, dim, dtype, more)
    desc = B.attention_packed(q0[-1], 12, 4, 1, dim, dtype=dtype, k_tokens=k0[-1])
    first = None
    for _ in range(20):
        o = torch.full_like(q, 7.0)
        launch(desc, [q, k, v, ints(q0), ints(k0), o])
        for s in range(12):
            assert not o[q0[s]:q0[s] + ql[s] - kl[s]].any()
        first = o if first is None else first
        assert torch.equal(o, first)
    some = slice(q0[11], q0[12])
    want, mag = dense(q[some], k[k0[11]:], v[k0[11]:], ql[11:], kl[11:], [0], [0], 1 / math.sqrt(dim))
    near(first[some], want, mag, DT[dtype])


def test_packed_attention_of_long_sequences_is_blind_to_keys_it_does_not_see():
    lens = [900, 1000, 800]
    q, k, v, q0, k0 = packed_case(lens, lens, 2, 1, 128, "bfloat16", 21)
    clean = [x.clone() for x in (q, k, v)]
    at = q0[1] + 700                                      # in the second tile of its pair
    v[at, 0, 3], v[at + 1, 0, 100] = float("nan"), -float("inf")
    v[q0[1] - 1, 0, 7], k[q0[1] - 1, 0, 7] = float("inf"), float("nan")   # the last key of the first sequence
    o = torch.zeros_like(q)
    launch(B.attention_packed(q0[-1], 3, 2, 1), [q, k, v, ints(q0), o])
    want, mag = dense(*clean, lens, lens, q0, k0, 1 / math.sqrt(128))
    fine = torch.ones(q0[-1], dtype=torch.bool, device="cuda")
    fine[q0[1] - 1] = False
    fine[at:q0[2]] = False
    near(o[fine], want[fine], mag[fine], torch.bfloat16)
    assert o[q0[1] - 1].isnan().all() and o[at:q0[2], :, 3].isnan().all()
    assert o[at, :, 100].isfinite().all() and bool((o[at + 1:at + 40, :, 100] == -math.inf).all())


def test_packed_attention_leaves_rows_outside_every_sequence():
    lens = [100, 260]
    q, k, v, q0, k0 = packed_case(lens, lens, 4, 4, 128, "bfloat16", 5, gap=37, tail=90)
    for x in (q, k, v):                                   # what lies there may be anything
        x[:37], x[397:] = float("nan"), float("inf")
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(q.shape[0], 2, 4, 4), [q, k, v, ints(q0), o])
    want, mag = dense(q, k, v, lens, lens, q0, k0, 1 / math.sqrt(128))
    near(o[37:397], want[37:397], mag[37:397], torch.bfloat16)
    assert bool((o[:37] == 7).all()) and bool((o[397:] == 7).all())


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 128), ("float16", 64)])
def test_packed_attention_is_blind_to_keys_it_does_not_see(dtype, dim):
    """Infinities and NaN in later keys and in other sequences do not reach a row; in keys it sees they do."""
    lens = [70, 300, 200]
    q, k, v, q0, k0 = packed_case(lens, lens, 2, 1, dim, dtype, 11)
    clean = [x.clone() for x in (q, k, v)]
    at = q0[1] + 150
    v[at, 0, 3], v[at + 1, 0, 5], v[at + 2, 0, 5], v[at + 3, 0, dim - 1] = float("nan"), float("inf"), -float("inf"), -float("inf")
    k[at + 20, 0, 1] = float("nan")
    q[q0[2] + 5, 0] = float("inf")
    o = torch.zeros_like(q)
    launch(B.attention_packed(q0[-1], 3, 2, 1, dim, dtype=dtype), [q, k, v, ints(q0), o])
    want, mag = dense(*clean, lens, lens, q0, k0, 1 / math.sqrt(dim))
    fine = torch.ones(q0[-1], 2, dtype=torch.bool, device="cuda")
    fine[at:q0[2]] = False
    fine[q0[2] + 5, 0] = False
    near(o[fine], want[fine], mag[fine], DT[dtype])
    rows = o[at:at + 20].float()                          # from the first bad value to the bad key
    assert rows[:, :, 3].isnan().all()
    assert bool((rows[1, :, 5] == math.inf).all()) and rows[2:, :, 5].isnan().all() and bool((rows[3:, :, dim - 1] == -math.inf).all())
    others = [d for d in range(dim) if d not in (3, 5, dim - 1)]
    near(o[at:at + 20][:, :, others], want[at:at + 20][:, :, others], mag[at:at + 20][:, :, others], DT[dtype])
    assert rows[0, :, 5].isfinite().all() and o[at + 20:q0[2]].isnan().all() and o[q0[2] + 5, 0].isnan().all()


@pytest.mark.parametrize("scale", [1e-3, 1.0, 40.0])
def test_packed_attention_of_flat_and_peaked_rows(scale):
    """Equal weights, and rows that one key takes whole (its reference moves often).  At scale 40 a score is up to 40 * 60 with an
    error of 2^-20 of 40 * 100 absolute products, 2^-8: the rows' weights are then known to 2^-7 only, which the bound gets."""
    q, k, v, q0, k0 = packed_case([700], [700], 2, 1, 128, "bfloat16", 3)
    o = torch.zeros_like(q)
    launch(B.attention_packed(700, 1, 2, 1, scale=scale), [q, k, v, ints(q0), o])
    want, mag = dense(q, k, v, [700], [700], q0, k0, scale)
    near(o, want, mag * (1 if scale <= 1 else 3), torch.bfloat16, f"scale {scale}")


def test_packed_attention_of_scores_far_below_zero():
    """Rows whose every score is -2^27 have equal weights, whatever a mask's lowest value may be elsewhere."""
    q, k, v, q0, k0 = packed_case([200], [200], 1, 1, 64, "bfloat16", 4)
    q.fill_(-2.0 ** 12)
    k.fill_(2.0 ** 12)
    o = torch.zeros_like(q)
    launch(B.attention_packed(200, 1, 1, 1, 64), [q, k, v, ints(q0), o])
    near(o, *dense(q, k, v, [200], [200], q0, k0, 1 / 8), torch.bfloat16)


def test_packed_attention_of_one_long_prompt():
    n = 20001
    q, k, v, q0, _ = packed_case([n], [n], 1, 1, 128, "bfloat16", 6)
    o = torch.zeros_like(q)
    launch(B.attention_packed(n, 1, 1, 1), [q, k, v, ints(q0), o])
    for row in (0, 127, 128, 9999, n - 2, n - 1):
        p = torch.softmax(q[row, 0].double() @ k[:row + 1, 0].double().T / math.sqrt(128), 0)
        near(o[row, 0], p @ v[:row + 1, 0].double(), p @ v[:row + 1, 0].double().abs(), torch.bfloat16, f"row {row}")


@pytest.mark.parametrize("layout", ["fused", "head_major"])
def test_packed_attention_layouts_agree_bit_for_bit(layout):
    lens, hq, hkv = [130, 5, 259], 8, 2
    q, k, v, q0, _ = packed_case(lens, lens, hq, hkv, 128, "bfloat16", 8)
    n, a = q0[-1], torch.zeros_like(q)
    launch(B.attention_packed(n, 3, hq, hkv), [q, k, v, ints(q0), a])
    b = torch.zeros_like(q)
    if layout == "fused":
        launch(B.attention_packed(n, 3, hq, hkv, fused=True), [torch.cat([q, k, v], 1).contiguous(), ints(q0), b])
    else:
        heads = [x.transpose(0, 1).contiguous() for x in (q, k, v, b)]
        launch(B.attention_packed(n, 3, hq, hkv, head_major=True), [*heads[:3], ints(q0), heads[3]])
        b = heads[3].transpose(0, 1)
    assert torch.equal(a, b)


def test_packed_attention_of_many_sequences():
    lens = [(7 * i) % 5 for i in range(D.PACKED_SEQS)]
    q, k, v, q0, k0 = packed_case(lens, lens, 1, 1, 64, "bfloat16", 9)
    o = torch.zeros_like(q)
    launch(B.attention_packed(q0[-1], len(lens), 1, 1, 64), [q, k, v, ints(q0), o])
    some = [i for i in range(len(lens)) if i % 97 == 0 or i > len(lens) - 6]
    want, mag = dense(q, k, v, [lens[i] for i in some], [lens[i] for i in some], [q0[i] for i in some], [k0[i] for i in some], 1 / 8)
    rows = [r for i in some for r in range(q0[i], q0[i + 1])]
    near(o[rows], want[rows], mag[rows], torch.bfloat16)


@pytest.mark.parametrize("table", [[0, 50, 40, 100], [0, 50, 60, 101], [-1, 50, 60, 100]])
def test_packed_attention_reports_a_bad_table(table):
    """The sequence with the bad entries is skipped, the others are computed."""
    q, k, v, _, _ = packed_case([100], [100], 2, 1, 64, "bfloat16", 10)
    o = torch.full_like(q, 7.0)
    assert failed(B.attention_packed(100, 3, 2, 1, 64), [q, k, v, ints(table), o]) == D.E_OOB
    if table[0] == 0:
        want, mag = dense(q, k, v, [50], [50], [0], [0], 1 / 8)
        near(o[:40], want[:40], mag[:40], torch.bfloat16)


def test_packed_attention_of_nothing():
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    launch(B.attention_packed(0, 2, 2, 2, 64), [q, q, q, ints([0, 0, 0]), q])
    q, k, v, q0, _ = packed_case([3], [3], 2, 1, 64, "bfloat16", 12)
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(3, 0, 2, 1, 64), [q, k, v, ints([0]), o])
    assert bool((o == 7).all())


# --------------------------------------------------------------------------------------------------------------------
# The 4-bit cache
# --------------------------------------------------------------------------------------------------------------------
def cache_case(lens, dim, page, group, hkv, dtype, seed, layers=1, spare=2):
    """A shape, a table of shuffled pages and an empty pool of a recognisable byte."""
    g = gen(seed)
    held = [-(-n // page) for n in lens]
    width, pages = max(1, max(held)), sum(held) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    c = B.kv4_cache(slots=len(lens), max_pages=width, pages=pages, hkv=hkv, dim=dim, page_size=page, group=group, layers=layers, dtype=dtype)
    return c, table, torch.full((c.pool_bytes,), 0xA5, dtype=torch.uint8, device="cuda")


def rows_of(n, c, seed, spread=1.0):
    g = gen(seed)
    return [(torch.randn(n, c.hkv, c.dim, generator=g) * spread + x).to(DT[c.dtype]).cuda() for x in (0.5, -0.25)]


SHAPES = [(128, 16, 64, 2, "bfloat16"), (128, 16, 32, 1, "float16"), (128, 32, 128, 3, "bfloat16"), (128, 64, 64, 1, "float16"),
          (128, 128, 32, 1, "bfloat16"), (64, 16, 64, 3, "float16"), (64, 32, 32, 1, "bfloat16"), (64, 128, 64, 2, "bfloat16")]


@pytest.mark.parametrize("dim,page,group,hkv,dtype", SHAPES)
def test_store_writes_the_defined_bytes_and_load_reads_them(dim, page, group, hkv, dtype):
    new, old = [1, 0, page + 3, 7], [page - 1, 4, 5, 0]              # across a page's end, none, several pages, a fresh slot
    lens = [a + b for a, b in zip(new, old)]
    c, table, pool = cache_case(lens, dim, page, group, hkv, dtype, page + dim, layers=2)
    k, v = rows_of(sum(new), c, 3)
    k[0, 0, :group] = 1.5                                            # a constant group
    v[1, 0, 0] = float("nan")
    k[2, 0, dim - 1] = -float("inf")
    want = S.Cache(c, pool.cpu(), table, lens)
    row = 0
    for s in range(4):
        for i in range(new[s]):
            for h in range(hkv):
                want.write(s, old[s] + i, h, k[row, h].cpu(), v[row, h].cpu(), layer=1)
            row += 1
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(new), layer=1), [k, v, ints(starts(new))] + books)
    got = pool.cpu().view(want.pool.shape)
    bad = (got != want.pool).nonzero()
    # A NaN's bits are free: compare those parameters by what they stand for, everything else by its bytes.
    back = S.Cache(c, pool.cpu(), table, lens)
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    launch(B.kv4_load(c, sum(new), layer=1), [ints(starts(new))] + books + [kb, vb])
    row = 0
    for s in range(4):
        for i in range(new[s]):
            for h in range(hkv):
                for x, y, z in zip(back.read(s, old[s] + i, h, 1), want.read(s, old[s] + i, h, 1), (kb, vb)):
                    assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(0), y.nan_to_num(0))
                    z = z[row, h].cpu().double()
                    assert torch.equal(z.isnan(), y.isnan())
                    y = y.nan_to_num(0)
                    lim = torch.finfo(DT[dtype]).eps / 2 * y.abs() + 2.0 ** -24 * 64 + SMALLEST[DT[dtype]]
                    assert bool(((z.nan_to_num(0) - y).abs() <= lim).all())
            row += 1
    assert len(bad) <= 8, f"{len(bad)} bytes differ from the definition"     # at most the two NaN pairs
    assert bool((got[0] == 0xA5).all())                                       # the other layer


@pytest.mark.parametrize("dim,group,hkv,dtype,page", [(128, 64, 5, "bfloat16", 16), (128, 32, 4, "float16", 64), (64, 32, 3, "bfloat16", 32),
                                                        (128, 64, 9, "bfloat16", 16), (64, 64, 17, "float16", 128), (128, 128, 2, "bfloat16", 64)])
def test_store_of_many_tokens_is_the_store_of_few(dim, group, hkv, dtype, page):
    """Several heads a warp (many tokens) and one (few) write the same bytes; the values are those of the definition."""
    lens = [4000, 1, 5100, 777]
    c, table, pool = cache_case(lens, dim, page, group, hkv, dtype, 3)
    k, v = rows_of(sum(lens), c, 4)
    cu, books = starts(lens), [ints(lens), ints(table)]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(cu)] + books + [pool])
    other, step = torch.full_like(pool, 0xA5), 500
    for s, n in enumerate(lens):
        for lo in range(0, n, step):
            m = min(step, n - lo)
            part = [0] * 4
            part[s] = m
            now = [lo + m if i == s else 0 for i in range(4)]
            rows = slice(cu[s] + lo, cu[s] + lo + m)
            launch(B.kv4_store(c, m), [k[rows], v[rows], ints(starts(part)), ints(now), ints(table), other])
    assert torch.equal(pool, other)
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    launch(B.kv4_load(c, sum(lens)), [ints(cu)] + books + [pool, kb, vb])
    for got, x in ((kb, k), (vb, v)):
        want = S.dequantised(x, group)
        lim = torch.finfo(DT[dtype]).eps / 2 * want.abs() + 2.0 ** -24 * 64 + SMALLEST[DT[dtype]]
        assert bool(((got.double() - want).abs() <= lim).all())


@pytest.mark.parametrize("dim,group", [(128, 64), (128, 32), (64, 64)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_codes_at_ties_and_at_the_ends_of_the_range(dim, group, dtype):
    """Values halfway between codes, exponents far apart, the smallest and the largest groups: each code is the defined one, so
    that what is read back is scale * code + minimum, one fp32 operation rounded once to the type."""
    t, r, n = DT[dtype], gen(91), 600
    low, high = (-126, 125) if dtype == "bfloat16" else (-14, 11)
    grid = torch.randint(0, 31, (n, 2, dim), generator=r).double() * 0.5
    grid.unflatten(-1, (-1, group))[..., 0], grid.unflatten(-1, (-1, group))[..., 1] = 0, 15   # the step is a power of two, ties abound
    grid = grid * 2.0 ** torch.randint(low + 1, high - 4, (n, 2, 1), generator=r).double()
    sign = torch.randint(0, 2, (n, 2, dim), generator=r).double() * 2 - 1
    apart = sign * 2.0 ** (torch.rand(n, 2, dim, generator=r).double() * 30 - 20).clamp(low, high)
    top = (torch.rand(n, 2, dim, generator=r).double() * 2 - 1) * torch.finfo(t).max
    tiny = torch.randint(-400, 400, (n, 2, dim), generator=r).double() * torch.finfo(t).smallest_normal * torch.finfo(t).eps
    edge = torch.rand(n, 2, dim, generator=r).double() * (15 if dtype == "bfloat16" else 1) * (1e-30 if dtype == "bfloat16" else 9e-4)
    x = torch.cat([grid, apart, top, tiny, edge]).to(t)
    c, table, pool = cache_case([5 * n], dim, 32, group, 2, dtype, 3)
    books = [ints([0, 5 * n]), ints([5 * n]), ints(table), pool]
    k, v = x.cuda(), x.flip(0).contiguous().cuda()
    launch(B.kv4_store(c, 5 * n), [k, v] + books)
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    launch(B.kv4_load(c, 5 * n), books + [kb, vb])
    for got, put in ((kb.cpu(), k.cpu()), (vb.cpu(), v.cpu())):
        code, scale, mn = S.quantise(put, group)
        want = code.unflatten(-1, (-1, group)).double() * scale.double()[..., None] + mn.double()[..., None]
        assert torch.equal(got, want.flatten(-2).float().to(t))


def test_a_cache_past_four_gigabytes():
    """Pages whose records lie past 2^32 bytes: written, read, attended to, and moved."""
    pages, lens = 300000, [33, 20]
    c = B.kv4_cache(slots=2, max_pages=3, pages=pages, hkv=8, dim=128, page_size=16, group=64)
    assert c.pool_bytes > 5 << 30
    pool = torch.empty(c.pool_bytes, dtype=torch.uint8, device="cuda")
    table = [[pages - 1, 7, pages - 5], [pages - 2, 250000, -1]]
    k, v = rows_of(53, c, 5)
    q = torch.randn(2, 16, 128, generator=gen(6)).to(torch.bfloat16).cuda()
    t, n, cu = ints(table), ints(lens), ints(starts(lens))
    launch(B.kv4_store(c, 53), [k, v, cu, n, t, pool])
    want, mag = cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128))
    o = torch.zeros_like(q)
    launch(B.attention_kv4(c, 16), [q, n, t, pool, o])
    near(o, want, mag, torch.bfloat16)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[[p for row in table for p in row if p >= 0]] = 1
    launch(B.pages_compact(c), [t, n, refs, pool])
    # used: 7, 250000, pages - 5, - 2, - 1; the k-th of those past 5 goes to the k-th free page below it
    assert t.tolist() == [[4, 0, 2], [3, 1, -1]]
    again = torch.zeros_like(q)
    launch(B.attention_kv4(c, 16), [q, n, t, pool, again])
    assert torch.equal(o, again)


def test_store_and_load_skip_and_report_what_has_no_place():
    lens = [20, 20, 40, 5]
    c, table, pool = cache_case(lens, 128, 16, 64, 1, "bfloat16", 1)
    k, v = rows_of(12, c, 5)
    table[1][1] = c.pages                                       # a page outside the pool
    table[2][2] = -1
    lens[3] = -2                                                # a length that cannot be
    before = pool.clone()
    cu, books = ints([0, 3, 6, 9, 12]), [ints(lens), ints(table), pool]
    assert failed(B.kv4_store(c, 12), [k, v, cu] + books) == D.E_OOB
    changed = (pool != before).view(c.pages, -1).any(1).nonzero().flatten().tolist()
    assert changed == [table[0][1]]
    kb, vb = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    assert failed(B.kv4_load(c, 12), [cu] + books + [kb, vb]) == D.E_OOB
    assert not kb[3:12].any() and not vb[3:12].any() and kb[:3].any()
    # rows outside every slot are left alone
    kb.fill_(3.0)
    launch(B.kv4_load(c, 12), [ints([2, 4, 4, 4, 4])] + books + [kb, vb])
    assert bool((kb[:2] == 3).all()) and bool((kb[4:] == 3).all()) and bool((kb[2:4] != 3).any())


def test_store_takes_a_fused_projection_and_head_major_keys():
    new = [5, 18]
    c, table, pool = cache_case(new, 128, 16, 64, 2, "bfloat16", 2)
    k, v = rows_of(23, c, 6)
    other = [pool.clone(), pool.clone()]
    cu, books = ints(starts(new)), [ints(new), ints(table)]
    launch(B.kv4_store(c, 23), [k, v, cu] + books + [pool])
    q = torch.randn(23, 6, 128, device="cuda").to(torch.bfloat16)
    launch(B.kv4_store(c, 23, fused_hq=6), [torch.cat([q, k, v], 1).contiguous(), cu] + books + [other[0]])
    launch(B.kv4_store(c, 23, head_major=True), [k.transpose(0, 1).contiguous(), v, cu] + books + [other[1]])
    assert torch.equal(pool, other[0]) and torch.equal(pool, other[1])


def cache_attention(q, k, v, lens, group, scale):
    """(o, bound on the weights' rounding / (eps / 2)) in float64, from the dense rows of each slot."""
    per = q.shape[1] // k.shape[1]
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    at = starts(lens)
    for s, n in enumerate(lens):
        for h in range(k.shape[1] if n else 0):
            kk, vv = (S.dequantised(x[at[s]:at[s + 1], h], group) for x in (k, v))
            a = S.quantise(v[at[s]:at[s + 1], h], group)[1].double().repeat_interleave(group, -1)
            rows = slice(h * per, (h + 1) * per)
            p = torch.softmax(q[s, rows].double() @ kk.T * scale, 1)
            out[s, rows], mag[s, rows] = p @ vv, 8 * (p @ a) + 0 * (p @ vv)
    return out, mag


ATTN = [(128, 16, 64, 2, 4, "bfloat16"), (128, 16, 32, 1, 8, "float16"), (128, 32, 128, 2, 1, "bfloat16"), (128, 64, 64, 1, 9, "float16"),
        (128, 128, 32, 1, 16, "bfloat16"), (64, 16, 64, 3, 3, "float16"), (64, 32, 32, 1, 17, "bfloat16"), (64, 128, 64, 2, 40, "bfloat16"),
        (128, 32, 64, 1, 12, "bfloat16")]
CONTEXTS = [[1], [0], [31, 0, 32, 33, 1, 16, 17, 64], [1000, 3, 129], [15] * 70]


@pytest.mark.parametrize("dim,page,group,hkv,per,dtype", ATTN)
@pytest.mark.parametrize("lens", CONTEXTS, ids=lambda x: str(x[:9]))
def test_cache_attention(dim, page, group, hkv, per, dtype, lens):
    c, table, pool = cache_case(lens, dim, page, group, hkv, dtype, sum(lens) + page)
    k, v = rows_of(sum(lens), c, 8)
    q = torch.randn(len(lens), hkv * per, dim, generator=gen(9)).to(DT[dtype]).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    o = torch.full_like(q, 7.0)
    launch(B.attention_kv4(c, hkv * per), [q] + books + [o])
    want, mag = cache_attention(q, k, v, lens, group, 1 / math.sqrt(dim))
    near(o, want, mag, DT[dtype])
    for s, n in enumerate(lens):
        assert n or not o[s].any()


@pytest.mark.parametrize("slots,dim,group,dtype", [(129, 128, 64, "bfloat16"), (464, 128, 64, "bfloat16"), (600, 128, 64, "bfloat16"),
                                                   (600, 64, 32, "float16"), (4096, 128, 32, "bfloat16"), (4096, 64, 64, "float16")])
def test_cache_attention_of_many_slots(slots, dim, group, dtype):
    """More slots than a CTA has threads: each sums a run of them.  Some hold nothing, runs of empty ones among them."""
    lens = [(37 * i * i + 11 * i) % 150 if i % 50 < 45 else 0 for i in range(slots)]
    c, table, pool = cache_case(lens, dim, 16, group, 1, dtype, slots)
    k, v = rows_of(sum(lens), c, 24)
    q = torch.randn(slots, 3, dim, generator=gen(25)).to(DT[dtype]).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    o = torch.full_like(q, 7.0)
    launch(B.attention_kv4(c, 3), [q] + books + [o])
    some = [s for s in range(slots) if s % 41 == 0 or s > slots - 60]
    at = starts(lens)
    rows = [r for s in some for r in range(at[s], at[s + 1])]
    near(o[some], *cache_attention(q[some], k[rows], v[rows], [lens[s] for s in some], group, 1 / math.sqrt(dim)), DT[dtype])
    assert not o[[s for s in range(slots) if not lens[s]]].any() and bool((o != 7).all())


@pytest.mark.parametrize("dtype,page", [("bfloat16", 16), ("float16", 64)])
def test_cache_attention_of_a_long_context(dtype, page):
    """100000 keys, whose weights average out: the result is 2^-8 of the values, and its error has to follow."""
    lens = [100001, 40]
    c, table, pool = cache_case(lens, 128, page, 64, 1, dtype, 4)
    k, v = rows_of(sum(lens), c, 10)
    v += 0.25                                                  # about zero
    q = torch.randn(2, 4, 128, generator=gen(11)).to(DT[dtype]).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    o = torch.zeros_like(q)
    launch(B.attention_kv4(c, 4), [q] + books + [o])
    want, mag = cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128))
    near(o, want, mag, DT[dtype])
    rel = (o.double() - want)[0].norm() / want[0].norm()
    # Independent roundings: each weight's is uniform within half a step, 1 / sqrt(3) of it on average, and meets a code whose distance
    # from 8 averages like the values themselves; the result's own rounding is the same size.  Four times their sum.
    assert rel < 4 * torch.finfo(DT[dtype]).eps / math.sqrt(3), rel


def test_cache_attention_ignores_what_lies_behind_a_slot():
    """The rest of the last page, other pages and a forked neighbour hold NaN parameters."""
    lens = [33, 5]
    for page in (16, 32, 64):
        c, table, pool = cache_case(lens, 128, page, 64, 2, "bfloat16", page)
        pool.fill_(0xFF)                                       # every parameter a NaN
        k, v = rows_of(sum(lens), c, 12)
        q = torch.randn(2, 8, 128, generator=gen(13)).to(torch.bfloat16).cuda()
        books = [ints(lens), ints(table), pool]
        launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
        o = torch.zeros_like(q)
        launch(B.attention_kv4(c, 8), [q] + books + [o])
        near(o, *cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128)), torch.bfloat16)


def test_cache_attention_passes_on_non_finite_keys_and_values_it_sees():
    lens = [40, 40, 40]
    c, table, pool = cache_case(lens, 64, 16, 32, 1, "bfloat16", 5)
    k, v = rows_of(120, c, 14)
    k[10, 0, 0] = float("nan")
    v[50, 0, 40] = float("inf")
    q = torch.randn(3, 2, 64, generator=gen(15)).to(torch.bfloat16).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, 120), [k, v, ints(starts(lens))] + books)
    o = torch.zeros_like(q)
    launch(B.attention_kv4(c, 2), [q] + books + [o])
    want, mag = cache_attention(q, k, v, lens, 32, 1 / 8)
    assert o[0].isnan().all() and o[1, :, 32:].isnan().all()
    near(o[1, :, :32], want[1, :, :32], mag[1, :, :32], torch.bfloat16)
    near(o[2], want[2], mag[2], torch.bfloat16)


@pytest.mark.parametrize("page,dtype", [(16, "bfloat16"), (64, "float16")])
def test_cache_attention_of_flat_and_peaked_rows(page, dtype):
    lens = [700, 65]
    c, table, pool = cache_case(lens, 128, page, 64, 1, dtype, 6)
    k, v = rows_of(sum(lens), c, 16)
    q = torch.randn(2, 8, 128, generator=gen(17)).to(DT[dtype]).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    for scale in (1e-4, 1.0):
        o = torch.zeros_like(q)
        launch(B.attention_kv4(c, 8, scale=scale), [q] + books + [o])
        near(o, *cache_attention(q, k, v, lens, 64, scale), DT[dtype], f"scale {scale}")


@pytest.mark.parametrize("dtype,power", [("float16", -14), ("float16", 8), ("bfloat16", -100), ("bfloat16", 100)])
def test_cache_attention_of_queries_far_from_one(dtype, power):
    """Queries at the ends of their type's range (fp16: 2^-14 times the usual, partly subnormal), the scale making up for it: the
    products are exact in powers of two, so the bound is that of usual queries."""
    lens = [700, 65]
    c, table, pool = cache_case(lens, 128, 16, 64, 1, dtype, 32)
    k, v = rows_of(sum(lens), c, 33)
    q = (torch.randn(2, 8, 128, generator=gen(34)) * 2.0 ** power).to(DT[dtype]).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    o = torch.zeros_like(q)
    scale = 2.0 ** -power / math.sqrt(128)
    launch(B.attention_kv4(c, 8, scale=scale), [q] + books + [o])
    near(o, *cache_attention(q, k, v, lens, 64, scale), DT[dtype])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("size", [1.0, 0.02, 1e-3, 1e-4])
@pytest.mark.parametrize("above,top", [(9, 0), (14, 0), (14, 1), (20, 0), (-20, 500)])
def test_cache_attention_of_small_values_behind_one_key(dtype, size, above, top):
    """One key's score `above` the others', its values `top` times theirs (-20, 500: far larger values with next to no weight); the
    slots are as many as the launch has warps, so that each is one part.  A weight times a scale keeps fp16's digits down to 2^-24 of
    the largest scale and is rounded by 2^-35 of it behind, which meets |code - 8| <= 8; the weights add up to 1 and more."""
    n, slots, hkv, dim, some = 1100, 222, 8, 128, [0, 100, 221]
    lens = [n] * slots
    c, table, pool = cache_case(lens, dim, 64, 64, hkv, dtype, 30)
    g = torch.Generator("cuda").manual_seed(31)
    k = torch.randn(slots * n, hkv, dim, generator=g, device="cuda") * 0.5
    v = (torch.rand(slots * n, hkv, dim, generator=g, device="cuda") + 1) * size
    v *= torch.where(torch.arange(dim, device="cuda") % 2 == 0, 1.0, -1.0)
    q = torch.randn(slots, hkv, dim, generator=g, device="cuda")
    at = torch.arange(slots, device="cuda") * n + 3
    k[at] = q * (above * math.sqrt(dim) / (q * q).sum(-1, keepdim=True))
    v[at] *= top
    k, v, q = (x.to(DT[dtype]) for x in (k, v, q))
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, slots * n), [k, v, ints(starts(lens))] + books)
    o = torch.zeros_like(q)
    launch(B.attention_kv4(c, hkv), [q] + books + [o])
    rows = [r for s in some for r in range(s * n, s * n + n)]
    want, mag = cache_attention(q[some], k[rows], v[rows], [n] * 3, 64, 1 / math.sqrt(dim))
    largest = float(S.quantise(v[rows], 64)[1].double().max())
    near(o[some], want, mag + 8 * n * 2.0 ** -35 * largest / (torch.finfo(DT[dtype]).eps / 2), DT[dtype])


def test_cache_attention_of_wide_values_in_fp16():
    """V scales of thousands times weights: no operand leaves fp16."""
    lens = [90]
    c, table, pool = cache_case(lens, 128, 16, 64, 1, "float16", 7)
    k, v = rows_of(90, c, 18)
    v[:, :, ::2], v[:, :, 1::2] = -60000.0, 60000.0
    v[::3] *= 0.5
    q = (torch.randn(1, 8, 128, generator=gen(19)) * 4).to(torch.float16).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, 90), [k, v, ints([0, 90])] + books)
    o = torch.zeros_like(q)
    launch(B.attention_kv4(c, 8), [q] + books + [o])
    near(o, *cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128)), torch.float16)


def test_cache_attention_reports_bad_pages_and_lengths():
    """A page outside the pool is not attended to, a length outside the row gives zeros; other slots are computed."""
    lens = [40, 40, 40]
    c, table, pool = cache_case(lens, 128, 16, 64, 1, "bfloat16", 8)
    k, v = rows_of(120, c, 20)
    q = torch.randn(3, 4, 128, generator=gen(21)).to(torch.bfloat16).cuda()
    launch(B.kv4_store(c, 120), [k, v, ints(starts(lens)), ints(lens), ints(table), pool])
    table[0][1] = -5                                            # keys 16 .. 31 of slot 0 are lost
    o = torch.zeros_like(q)
    assert failed(B.attention_kv4(c, 4), [q, ints([40, 49, 40]), ints(table), pool, o]) == D.E_OOB
    keep = [t for t in range(120) if not 16 <= t < 32]
    want, mag = cache_attention(q, k[keep], v[keep], [24, 40, 40], 64, 1 / math.sqrt(128))
    near(o[[0, 2]], want[[0, 2]], mag[[0, 2]], torch.bfloat16)
    assert not o[1].any()


def test_cache_attention_takes_a_fused_projection():
    lens = [50, 20]
    c, table, pool = cache_case(lens, 128, 16, 64, 2, "bfloat16", 9)
    k, v = rows_of(70, c, 22)
    q = torch.randn(2, 8, 128, generator=gen(23)).to(torch.bfloat16).cuda()
    books = [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, 70), [k, v, ints(starts(lens))] + books)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    launch(B.attention_kv4(c, 8), [q] + books + [a])
    launch(B.attention_kv4(c, 8, fused=True), [torch.cat([q, k[:2], v[:2]], 1).contiguous()] + books + [b])
    assert torch.equal(a, b)


def test_attention_without_any_key():
    """No key row at all, and a cache without pages: every query gives zeros."""
    q = torch.randn(200, 4, 64, generator=gen(93)).to(torch.bfloat16).cuda()
    none = torch.empty(0, dtype=torch.bfloat16, device="cuda")
    o = torch.full_like(q, 7.0)
    launch(B.attention_packed(200, 2, 4, 2, 64, k_tokens=0), [q, none, none, ints([0, 150, 200]), ints([0, 0, 0]), o])
    assert not o.any()
    c = B.kv4_cache(slots=3, max_pages=0, pages=0, hkv=2, dim=64)
    o = torch.full_like(q[:3], 7.0)
    launch(B.attention_kv4(c, 4), [q[:3].contiguous(), ints([0, 0, 0]), ints([]), torch.empty(0, dtype=torch.uint8, device="cuda"), o])
    assert not o.any()


# --------------------------------------------------------------------------------------------------------------------
# Page bookkeeping
# --------------------------------------------------------------------------------------------------------------------
class Live:
    """The device state beside the oracle's."""

    def __init__(self, slots=6, width=5, pages=23, page=16, layers=2, hkv=1):
        self.c = B.kv4_cache(slots=slots, max_pages=width, pages=pages, hkv=hkv, dim=64, page_size=page, group=64, layers=layers)
        self.table, self.lens, self.refs = ints([[-1] * width] * slots), ints([0] * slots), ints([0] * pages)
        self.pool = torch.randint(0, 256, (layers, pages, self.c.page_bytes), generator=gen(pages), dtype=torch.uint8).cuda()
        self.want = S.Pages(self.table.tolist(), [0] * slots, [0] * pages, self.pool.cpu(), page)

    def books(self):
        return [self.table, self.lens, self.refs]

    def same(self):
        assert self.table.tolist() == self.want.table and self.lens.tolist() == self.want.lens
        assert self.refs.tolist() == self.want.refs and torch.equal(self.pool.cpu(), self.want.pool)

    def grow(self, ids, add):
        launch(B.pages_grow(self.c, len(ids)), [ints(ids), ints(add)] + self.books())
        self.want.grow(ids, add)
        self.same()

    def fork(self, src, dst, deep=False):
        launch(B.pages_fork(self.c, len(src), deep), [ints(src), ints(dst)] + self.books() + [self.pool])
        self.want.fork(src, dst, deep)
        self.same()

    def free(self, ids):
        launch(B.pages_free(self.c, len(ids)), [ints(ids)] + self.books())
        self.want.free(ids)
        self.same()

    def compact(self):
        launch(B.pages_compact(self.c), self.books() + [self.pool])
        self.want.compact()
        self.same()


def test_pages_by_hand():
    a = Live()
    a.grow([2, 0], [17, 16])                  # two pages, one page
    a.grow([0, 2, 1], [0, 15, 1])             # nothing, to the end of a page, a fresh slot
    a.fork([2, 0], [3, 4])                    # full pages only: nothing is copied
    a.grow([2, 0], [1, 3])                    # past the shared pages: pages of their own
    a.fork([2], [5])
    a.free([2, 1, 2])                         # one slot listed twice
    a.compact()
    a.compact()                               # nothing to move
    a.fork([5, 0], [1, 2], deep=True)
    a.free([5, 4, 3, 0])
    a.compact()
    a.free([1, 2])
    assert not a.refs.any()


@pytest.mark.parametrize("slots,width,pages,page", [(6, 5, 23, 16), (40, 3, 90, 32), (9, 700, 5001, 16), (300, 60, 16400, 16)])
def test_pages_at_random(slots, width, pages, page):
    """Any order of operations that fits, against the slot-by-slot bookkeeping."""
    import random
    rng = random.Random(slots)
    a = Live(slots, width, pages, page)
    for _ in range(14):
        room = sum(r <= 0 for r in a.want.refs)
        empty = [s for s in range(slots) if not a.want.lens[s]]
        full = [s for s in range(slots) if a.want.lens[s]]
        what = rng.choice(["grow", "grow", "fork", "copy", "free", "compact"])
        if what == "grow":
            ids = rng.sample(range(slots), rng.randint(1, slots))
            add = [rng.randint(0, max(0, min(width * page - a.want.lens[s], max(0, room // len(ids) - 1) * page))) for s in ids]
            a.grow(ids, add)
        elif what in ("fork", "copy") and full and empty:
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(full) for _ in dst]
            while dst and sum(a.want.held(a.want.lens[s]) if what == "copy" else 1 for s in src) > room:
                src, dst = src[:-1], dst[:-1]
            if dst:
                a.fork(src, dst, what == "copy")
        elif what == "free" and full:
            a.free([rng.choice(full) for _ in range(rng.randint(1, len(full)))])
        else:
            a.compact()


def test_pages_refuse_and_leave_everything_as_it_was():
    a = Live(slots=5, width=4, pages=7, page=16)
    a.grow([0, 1], [40, 20])                  # 3 + 2 pages of 7
    ops = [
        (B.pages_grow(a.c, 2), [[0, 5], [1, 1]], False, D.E_OOB),            # a slot outside
        (B.pages_grow(a.c, 2), [[0, -1], [1, 1]], False, D.E_OOB),
        (B.pages_grow(a.c, 2), [[2, 2], [1, 1]], False, D.E_ARGS),           # listed twice
        (B.pages_grow(a.c, 2), [[2, 3], [1, -1]], False, D.E_ARGS),
        (B.pages_grow(a.c, 2), [[2, 0], [1, 25]], False, D.E_RESOURCE),      # past the row
        (B.pages_grow(a.c, 2), [[2, 3], [17, 20]], False, D.E_RESOURCE),     # 4 pages of the 2 free ones
        (B.pages_grow(a.c, 2), [[2, 0], [1, 2 ** 31 - 1]], False, D.E_RESOURCE),
        (B.pages_fork(a.c, 2), [[0, 1], [2, 2]], True, D.E_ARGS),            # one target twice
        (B.pages_fork(a.c, 2), [[0, 0], [2, 1]], True, D.E_ARGS),            # a target in use
        (B.pages_fork(a.c, 2), [[0, 3], [3, 4]], True, D.E_ARGS),            # a target that is a source
        (B.pages_fork(a.c, 2), [[0, 1], [2, 7]], True, D.E_OOB),
        (B.pages_fork(a.c, 1, True), [[0], [2]], True, D.E_RESOURCE),        # 3 pages of 2
        (B.pages_free(a.c, 1), [[9]], False, D.E_OOB),
    ]
    for desc, lists, pool, code in ops:
        n = len(lists[0])
        assert failed(desc, [ints(x) for x in lists] + a.books() + ([a.pool] if pool else [])) == code, (lists, n)
        a.same()
    a.fork([0, 1], [2, 3])                    # the two partial pages take the two free ones
    assert failed(B.pages_fork(a.c, 1), [ints([0]), ints([4])] + a.books() + [a.pool]) == D.E_RESOURCE
    a.same()


# --------------------------------------------------------------------------------------------------------------------
# Together, and as programs use them
# --------------------------------------------------------------------------------------------------------------------
def test_a_serving_loop():
    """Prompts admitted, attended and stored, decoded in a batch, forked, decoded apart, freed and compacted: the cache holds what a
    dense history says at every step, and compaction changes no result."""
    hq, hkv, dim, page, group = 8, 2, 128, 16, 64
    c = B.kv4_cache(slots=5, max_pages=8, pages=24, hkv=hkv, dim=dim, page_size=page, group=group, layers=2)
    g = gen(31)
    table, lens, refs = ints([[-1] * 8] * 5), ints([0] * 5), ints([0] * 24)
    pool = torch.zeros(c.pool_bytes, dtype=torch.uint8, device="cuda")
    books, layer, scale = [table, lens, refs], 1, 1 / math.sqrt(dim)
    past = [[] for _ in range(5)]             # (k, v) rows of every slot, dense

    def project(n):
        return torch.randn(n, hq + 2 * hkv, dim, generator=g).to(torch.bfloat16).cuda()

    def admit(new):
        """new: {slot: prompt length}."""
        ids = sorted(new)
        launch(B.pages_grow(c, len(ids)), [ints(ids), ints([new[s] for s in ids])] + books)
        counts = [new.get(s, 0) for s in range(5)]
        qkv, cu = project(sum(counts)), starts(counts)
        o = torch.zeros(sum(counts), hq, dim, dtype=torch.bfloat16, device="cuda")
        launch(B.attention_packed(sum(counts), 5, hq, hkv, fused=True), [qkv, ints(cu), o])
        launch(B.kv4_store(c, sum(counts), layer, fused_hq=hq), [qkv, ints(cu), lens, table, pool])
        q, k, v = (x.contiguous() for x in qkv.split([hq, hkv, hkv], 1))
        near(o, *dense(q, k, v, counts, counts, cu, cu, scale), torch.bfloat16)
        for s in ids:
            past[s] += [(k[t], v[t]) for t in range(cu[s], cu[s + 1])]

    def attend(q):
        o = torch.full((5, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        launch(B.attention_kv4(c, hq, layer), [q, lens, table, pool, o])
        return o

    def decode(ids):
        """One token for each of the slots `ids`; every slot attends."""
        launch(B.pages_grow(c, len(ids)), [ints(ids), ints([1] * len(ids))] + books)
        counts = [int(s in ids) for s in range(5)]
        qkv = project(len(ids))
        launch(B.kv4_store(c, len(ids), layer, fused_hq=hq), [qkv, ints(starts(counts)), lens, table, pool])
        for row, s in enumerate(sorted(ids)):
            past[s].append((qkv[row, hq:hq + hkv], qkv[row, hq + hkv:]))
        q = torch.randn(5, hq, dim, generator=g).to(torch.bfloat16).cuda()
        o = attend(q)
        n = [len(p) for p in past]
        assert lens.tolist() == n
        k, v = (torch.stack([kv[i] for p in past for kv in p]) for i in (0, 1))
        near(o, *cache_attention(q, k, v, n, group, scale), torch.bfloat16)
        return q, o

    admit({0: 37, 2: 16, 4: 1})
    for _ in range(3):
        decode([0, 2, 4])
    launch(B.pages_fork(c, 2), [ints([0, 0]), ints([1, 3])] + books + [pool])
    past[1], past[3] = list(past[0]), list(past[0])
    for _ in range(2):
        decode([0, 1, 2, 3, 4])               # the forks part ways
    launch(B.pages_free(c, 2), [ints([0, 2])] + books)
    past[0], past[2] = [], []
    q, before = decode([1, 4])
    launch(B.pages_compact(c), books + [pool])
    assert torch.equal(attend(q), before)
    admit({0: 90})
    decode([0, 1, 3, 4])
    live = int((refs > 0).sum())
    assert sorted(set(table.flatten().tolist()) - {-1}) == torch.nonzero(refs > 0).flatten().tolist() and live <= 24


def decode_graph(seed, slots=3):
    lens = [50, 7, 33][:slots]
    c, table, pool = cache_case(lens, 128, 16, 64, 2, "bfloat16", seed)
    k, v = rows_of(sum(lens), c, seed)
    q = torch.randn(slots, 8, 128, generator=gen(seed + 1)).to(torch.bfloat16).cuda()
    o = torch.zeros_like(q)
    books = [ints(lens), ints(table), pool]
    g = Graph("cuda:0")
    for n, t in zip(("k", "v", "cu", "lens", "table", "pool", "q", "o"), (k, v, ints(starts(lens)), *books, q, o)):
        g.bind(n, t)
    g.add("store", D.to_bytes(B.kv4_store(c, sum(lens))), ["k", "v", "cu", "lens", "table", "pool"])
    g.add("attend", D.to_bytes(B.attention_kv4(c, 8)), ["q", "lens", "table", "pool", "o"])
    return g, o, cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128))


def test_captured_graphs_replay_on_two_streams():
    """Two captured decode steps replayed at once share nothing; an eager run between them changes neither."""
    (a, oa, wa), (b, ob, wb) = decode_graph(40), decode_graph(50)
    a.capture(), b.capture()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    oa.zero_(), ob.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(sa):
            a.cuda_graph.replay()
        with torch.cuda.stream(sb):
            b.cuda_graph.replay()
    torch.cuda.synchronize()
    near(oa, *wa, torch.bfloat16)
    near(ob, *wb, torch.bfloat16)


def test_a_captured_decode_step_grows_its_slots():
    """Grow, store and attend as one replayed graph: the capture's own first run is a step, then each replay is one."""
    slots, hq, hkv = 4, 8, 2
    c = B.kv4_cache(slots=slots, max_pages=4, pages=16, hkv=hkv, dim=128, page_size=16, group=64)
    state = {"ids": ints([0, 1, 2, 3]), "one": ints([1] * 4), "table": ints([[-1] * 4] * 4), "lens": ints([0] * 4), "refs": ints([0] * 16),
             "pool": torch.zeros(c.pool_bytes, dtype=torch.uint8, device="cuda"), "cu": ints(range(5)),
             "qkv": torch.zeros(slots, hq + 2 * hkv, 128, dtype=torch.bfloat16, device="cuda"),
             "o": torch.zeros(slots, hq, 128, dtype=torch.bfloat16, device="cuda")}
    g = Graph("cuda:0")
    for name, t in state.items():
        g.bind(name, t)
    g.add("grow", D.to_bytes(B.pages_grow(c, slots)), ["ids", "one", "table", "lens", "refs"])
    g.add("store", D.to_bytes(B.kv4_store(c, slots, fused_hq=hq)), ["qkv", "cu", "lens", "table", "pool"])
    g.add("attend", D.to_bytes(B.attention_kv4(c, hq, fused=True)), ["qkv", "lens", "table", "pool", "o"])
    past, r = [], gen(90)
    for step in range(40):
        state["qkv"].copy_(torch.randn(slots, hq + 2 * hkv, 128, generator=r).to(torch.bfloat16))
        past.append(state["qkv"].clone())
        if step == 0:
            g.capture()
        else:
            g.run()
        if step in (0, 15, 16, 39):
            native.sync(torch.cuda.current_stream().cuda_stream)
            rows = torch.stack(past, 1).flatten(0, 1)          # slot by slot
            q, k, v = (x.contiguous() for x in rows.split([hq, hkv, hkv], 1))
            near(state["o"], *cache_attention(past[-1][:, :hq], k, v, [step + 1] * slots, 64, 1 / math.sqrt(128)), torch.bfloat16)
    assert state["lens"].tolist() == [40] * 4 and int((state["refs"] > 0).sum()) == 12


def test_a_captured_decode_step_that_runs_out_of_pages_leaves_the_cache():
    """Four slots of one page each and one page to spare: the step that needs four more is refused, and from there the replays change
    nothing; with a slot freed and the halt word cleared they go on, and every token is where the dense history has it."""
    slots, hq, hkv = 4, 8, 2
    c = B.kv4_cache(slots=slots, max_pages=4, pages=5, hkv=hkv, dim=128, page_size=16, group=64)
    state = {"ids": ints([0, 1, 2, 3]), "one": ints([1] * 4), "table": ints([[-1] * 4] * 4), "lens": ints([0] * 4), "refs": ints([0] * 5),
             "halt": ints([0]), "pool": torch.zeros(c.pool_bytes, dtype=torch.uint8, device="cuda"), "cu": ints(range(5)),
             "qkv": torch.zeros(slots, hq + 2 * hkv, 128, dtype=torch.bfloat16, device="cuda"),
             "o": torch.zeros(slots, hq, 128, dtype=torch.bfloat16, device="cuda")}
    g = Graph("cuda:0")
    for name, t in state.items():
        g.bind(name, t)
    g.add("grow", D.to_bytes(B.pages_grow(c, slots, halt=True)), ["ids", "one", "table", "lens", "refs", "halt"])
    g.add("store", D.to_bytes(B.kv4_store(c, slots, fused_hq=hq, halt=True)), ["qkv", "cu", "lens", "table", "pool", "halt"])
    g.add("attend", D.to_bytes(B.attention_kv4(c, hq, fused=True)), ["qkv", "lens", "table", "pool", "o"])
    past, r, stream = [], gen(91), torch.cuda.current_stream().cuda_stream

    def step():
        state["qkv"].copy_(torch.randn(slots, hq + 2 * hkv, 128, generator=r).to(torch.bfloat16))
        past.append(state["qkv"].clone())
        g.run() if g.cuda_graph else g.capture()

    for _ in range(16):
        step()
    native.sync(stream)
    books = [state[n].clone() for n in ("table", "lens", "refs", "pool")]
    for _ in range(3):                                       # refused once, then halted
        step()
    with pytest.raises(native.ExecutorError) as e:
        native.sync(stream)
    assert e.value.code == D.E_RESOURCE and state["halt"].tolist() == [D.E_RESOURCE]
    for t, n in zip(books, ("table", "lens", "refs", "pool")):
        assert torch.equal(t, state[n]), n
    del past[16:]
    for desc, ts in ((B.pages_free(c, 1, halt=True), [ints([3])] + [state[n] for n in ("table", "lens", "refs", "halt")]),
                     (B.kv4_store(c, 4, fused_hq=hq, halt=True), [state[n] for n in ("qkv", "cu", "lens", "table", "pool", "halt")])):
        assert failed(desc, ts) == D.E_RESOURCE              # halted as well, and each says so
        assert state["lens"].tolist() == [16] * 4 and torch.equal(books[3], state["pool"])
    launch(B.pages_free(c, 3), [ints([1, 2, 3])] + [state[n] for n in ("table", "lens", "refs")])
    state["halt"].zero_()
    step()
    native.sync(stream)
    assert state["lens"].tolist() == [17, 1, 1, 1]
    rows = torch.cat([torch.stack(past)[:, 0], past[-1][1:]])
    q, k, v = (x.contiguous() for x in rows.split([hq, hkv, hkv], 1))
    near(state["o"], *cache_attention(past[-1][:, :hq], k, v, [17, 1, 1, 1], 64, 1 / math.sqrt(128)), torch.bfloat16)


def test_a_failure_is_raised_by_the_next_synchronisation_and_once():
    """Of whichever operator: the launches after it run, and give what they always give."""
    a = Live(slots=2, width=2, pages=1, page=16)
    RC.launch_tensors(D.to_bytes(B.pages_grow(a.c, 1)), [ints([0]), ints([17])] + a.books(), sync=False)   # two pages of one
    q, k, v, q0, k0 = packed_case([40], [40], 2, 1, 64, "bfloat16", 92)
    o, again = torch.zeros_like(q), torch.zeros_like(q)
    blob = D.to_bytes(B.attention_packed(40, 1, 2, 1, 64))
    with pytest.raises(native.ExecutorError) as e:
        RC.launch_tensors(blob, [q, k, v, ints(q0), o])
    assert e.value.code == D.E_RESOURCE
    RC.launch_tensors(blob, [q, k, v, ints(q0), again])
    near(o, *dense(q, k, v, [40], [40], q0, k0, 1 / 8), torch.bfloat16)
    assert torch.equal(o, again)
    a.same()


def test_a_refused_fork_halts_what_follows():
    a = Live(slots=5, width=4, pages=7, page=16)
    a.grow([0, 1], [40, 20])                                 # 3 + 2 pages of 7
    halt = ints([0])
    lists = lambda *x: [ints(i) for i in x] + a.books()
    RC.launch_tensors(D.to_bytes(B.pages_fork(a.c, 1, deep=True, halt=True)), lists([0], [2]) + [a.pool, halt], sync=False)   # 3 pages of 2
    k, v = rows_of(2, a.c, 3)
    k, v = (x[:, :a.c.hkv].contiguous() for x in (k, v))
    for desc, ts in ((B.pages_fork(a.c, 1, halt=True), lists([1], [3]) + [a.pool, halt]), (B.pages_grow(a.c, 1, halt=True), lists([1], [1]) + [halt]),
                     (B.kv4_store(a.c, 2, halt=True), [k, v, ints([0, 1, 2, 2, 2, 2]), a.lens, a.table, a.pool.flatten(), halt]),
                     (B.pages_free(a.c, 2, halt=True), lists([0, 1]) + [halt]), (B.pages_compact(a.c, halt=True), a.books() + [a.pool, halt])):
        RC.launch_tensors(D.to_bytes(desc), ts, sync=False)
    with pytest.raises(native.ExecutorError) as e:
        native.sync(torch.cuda.current_stream().cuda_stream)
    assert e.value.code == D.E_RESOURCE and halt.tolist() == [D.E_RESOURCE]
    a.same()
    halt.zero_()
    launch(B.pages_fork(a.c, 1, halt=True), lists([1], [3]) + [a.pool, halt])
    a.want.fork([1], [3])
    a.same()
    assert not halt.any()


def test_launches_on_two_streams_do_not_share_a_workspace():
    def case(seed, n):
        c, table, pool = cache_case([n], 128, 16, 64, 1, "bfloat16", seed)
        k, v = rows_of(n, c, seed)
        q = torch.randn(1, 4, 128, generator=gen(seed)).to(torch.bfloat16).cuda()
        books = [ints([n]), ints(table), pool]
        launch(B.kv4_store(c, n), [k, v, ints([0, n])] + books)
        return D.to_bytes(B.attention_kv4(c, 4)), [q] + books + [torch.zeros_like(q)], cache_attention(q, k, v, [n], 64, 1 / math.sqrt(128))
    cases = [case(60, 6000), case(61, 9000)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for (blob, ts, _), s in zip(cases, streams):
            with torch.cuda.stream(s):
                RC.launch_tensors(blob, ts, sync=False)
    torch.cuda.synchronize()
    for _, ts, want in cases:
        near(ts[-1], *want, torch.bfloat16)


def test_launches_on_given_streams_have_workspaces_of_their_own():
    """`stream=` with another stream current: eager, and as two branches of one capture that run at the same time."""
    def case(seed, n):
        c, table, pool = cache_case([n], 128, 16, 64, 1, "bfloat16", seed)
        k, v = rows_of(n, c, seed)
        q = torch.randn(1, 4, 128, generator=gen(seed)).to(torch.bfloat16).cuda()
        books = [ints([n]), ints(table), pool]
        launch(B.kv4_store(c, n), [k, v, ints([0, n])] + books)
        return D.to_bytes(B.attention_kv4(c, 4)), [q] + books + [torch.zeros_like(q)], cache_attention(q, k, v, [n], 64, 1 / math.sqrt(128))
    cases = [case(62, 20000), case(63, 17000)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def both():
        for (blob, ts, _), s in zip(cases, streams):
            for _ in range(4):
                RC.launch_tensors(blob, ts, stream=s, sync=False)

    def right():
        torch.cuda.synchronize()
        for _, ts, want in cases:
            near(ts[-1], *want, torch.bfloat16)
            ts[-1].zero_()
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    both()
    right()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        both()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        g.replay()
        right()


def test_launch_tensors_can_be_captured():
    lens = [30, 200]
    q, k, v, q0, k0 = packed_case(lens, lens, 4, 2, 128, "bfloat16", 70)
    o = torch.zeros_like(q)
    a = Live()
    blobs = [(D.to_bytes(B.attention_packed(230, 2, 4, 2)), [q, k, v, ints(q0), o]),
             (D.to_bytes(B.pages_grow(a.c, 1)), [ints([1]), ints([20])] + a.books()),
             (D.to_bytes(B.pages_fork(a.c, 1)), [ints([1]), ints([3])] + a.books() + [a.pool]),
             (D.to_bytes(B.pages_free(a.c, 2)), [ints([1, 3])] + a.books())]
    for blob, ts in blobs:
        RC.launch_tensors(blob, ts)
    o.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for blob, ts in blobs:
            RC.launch_tensors(blob, ts, sync=False)
    for _ in range(3):
        g.replay()
    native.sync(torch.cuda.current_stream().cuda_stream)
    near(o, *dense(q, k, v, lens, lens, q0, k0, 1 / math.sqrt(128)), torch.bfloat16)
    assert not a.refs.any() and not a.lens.any()


@pytest.mark.parametrize("family", ["packed", "packed_long", "kv4"])
def test_stalled_stage_times_out_and_device_stays_usable(family):
    """A withheld copy ends in PTSIM_E_TIMEOUT within the test's limit, and the next launch is right."""
    if family != "kv4":
        lens = [600 if family == "packed" else 1600]
        q, k, v, q0, k0 = packed_case(lens, lens, 2, 1, 128, "bfloat16", 80)
        o = torch.zeros_like(q)
        desc, ts, want = B.attention_packed(lens[0], 1, 2, 1), [q, k, v, ints(q0), o], dense(q, k, v, lens, lens, q0, k0, 1 / math.sqrt(128))
    else:
        lens = [900]
        c, table, pool = cache_case(lens, 128, 16, 64, 1, "bfloat16", 81)
        k, v = rows_of(900, c, 82)
        q = torch.randn(1, 4, 128, generator=gen(83)).to(torch.bfloat16).cuda()
        o, books = torch.zeros_like(q), [ints(lens), ints(table), pool]
        launch(B.kv4_store(c, 900), [k, v, ints([0, 900])] + books)
        desc, ts, want = B.attention_kv4(c, 4), [q] + books + [o], cache_attention(q, k, v, lens, 64, 1 / math.sqrt(128))
    stalled = D.from_bytes(D.to_bytes(desc))
    stalled.flags |= D.FLAG_TEST_STALL
    assert failed(stalled, ts) == D.E_TIMEOUT
    launch(desc, ts)
    near(o, *want, torch.bfloat16)


@pytest.mark.parametrize("dim,group,per,dtype", [(128, 64, 4, "bfloat16"), (64, 32, 12, "float16"), (128, 32, 9, "bfloat16")])
def test_a_stalled_cache_tile_ends_its_own_part_only(dim, group, per, dtype):
    """The warp whose first tile never lands gives up as a whole: the slots that it holds nothing of are computed."""
    lens = [64] + [300] * 11
    c, table, pool = cache_case(lens, dim, 16, group, 1, dtype, 84)
    k, v = rows_of(sum(lens), c, 85)
    q = torch.randn(12, per, dim, generator=gen(86)).to(DT[dtype]).cuda()
    o, books = torch.full_like(q, 7.0), [ints(lens), ints(table), pool]
    launch(B.kv4_store(c, sum(lens)), [k, v, ints(starts(lens))] + books)
    stalled = B.attention_kv4(c, per)
    stalled.flags |= D.FLAG_TEST_STALL
    assert failed(stalled, [q] + books + [o]) == D.E_TIMEOUT
    want, mag = cache_attention(q, k, v, lens, group, 1 / math.sqrt(dim))
    near(o[1:], want[1:], mag[1:], DT[dtype])
    assert bool((o[0] == 7).all())
    launch(B.attention_kv4(c, per), [q] + books + [o])
    near(o, want, mag, DT[dtype])
