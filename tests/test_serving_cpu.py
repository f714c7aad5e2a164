"""The serving operators without a GPU: their descriptors and refusals (ptsim_check), their access streams, and the
64-bit oracle's own consistency (a token written into a record reads back as the values its codes stand for)."""
import contextlib
import json
import types

import pytest
import torch

from oracle import serving as S
from pytorchsim_triton_compiler.codegen import build as B
from pytorchsim_triton_compiler.codegen import descriptors as D
from pytorchsim_triton_compiler.runtime import cuda as RC
from pytorchsim_triton_compiler.runtime import dma_access, native
from pytorchsim_triton_compiler.runtime.graph import Graph

SHAPES = [(64, 16, 32, 2), (64, 32, 64, 1), (128, 16, 64, 2), (128, 64, 32, 1), (128, 128, 128, 1)]   # dim, page, group, hkv


def shape(dim=128, page=16, group=64, hkv=2, slots=3, max_pages=4, pages=9, layers=2, dtype="bfloat16"):
    return B.kv4_cache(slots=slots, max_pages=max_pages, pages=pages, hkv=hkv, dim=dim, page_size=page, group=group,
                       layers=layers, dtype=dtype)


def every_builder():
    c = shape()
    yield "packed", B.attention_packed(10, 3, 8, 2)
    yield "packed fused", B.attention_packed(10, 3, 8, 2, 64, dtype="float16", fused=True)
    yield "packed prefix", B.attention_packed(10, 3, 8, 2, k_tokens=21)
    yield "packed head major", B.attention_packed(10, 3, 8, 2, head_major=True)
    yield "store", B.kv4_store(c, 7, layer=1)
    yield "store fused", B.kv4_store(c, 7, fused_hq=4)
    yield "store head major", B.kv4_store(c, 7, head_major=True)
    yield "load", B.kv4_load(c, 7)
    yield "attention", B.attention_kv4(c, 6)
    yield "attention fused", B.attention_kv4(c, 6, fused=True)
    yield "grow", B.pages_grow(c, 2)
    yield "fork", B.pages_fork(c, 2)
    yield "copy", B.pages_fork(c, 2, deep=True)
    yield "free", B.pages_free(c, 2)
    yield "compact", B.pages_compact(c)


@pytest.mark.parametrize("name,desc", list(every_builder()), ids=lambda x: x if isinstance(x, str) else "")
def test_descriptors_validate_and_describe(name, desc):
    blob = D.to_bytes(desc)
    native.check(blob)
    assert native.units(blob) == 1
    assert D.describe(D.from_bytes(blob))["kind"] == D.SERVING_NAME[desc.kind]
    outs = RC.written_args(desc)
    names = [f"a{i}" for i in range(desc.nargs)]
    streams = dma_access.streams(desc, 0, 1, names)
    assert {s["arg"] for s in streams if s["dir"] == "write"} == {names[i] for i in outs}
    assert {s["arg"] for s in streams} == set(names)
    for s in streams:
        ends = dma_access.bounds(s["access"])
        if ends is not None:
            assert 0 <= ends[0] and ends[1] < desc.arg_numel[names.index(s["arg"])]


def _code(desc):
    with pytest.raises(native.ExecutorError) as e:
        native.check(D.to_bytes(desc))
    return e.value.code


def _with(desc, params, **fields):
    for k, v in fields.items():
        setattr(getattr(desc.p, params), k, v)
    return desc


@pytest.mark.parametrize("fields,code", [
    (dict(dim=96), D.E_UNSUPPORTED), (dict(hq=7), D.E_DESC), (dict(scale=0.0), D.E_UNSUPPORTED),
    (dict(scale=float("nan")), D.E_UNSUPPORTED), (dict(scale=float("inf")), D.E_UNSUPPORTED),
    (dict(q_tokens=11), D.E_OOB), (dict(k_tokens=11), D.E_OOB), (dict(q_off=4), D.E_UNSUPPORTED),
    (dict(k_row=2 * 128 + 4), D.E_UNSUPPORTED), (dict(o_row=-8), D.E_DESC), (dict(seqs=4), D.E_OOB), (dict(seqs=-1), D.E_DESC),
    (dict(seqs=D.PACKED_SEQS + 1), D.E_UNSUPPORTED), (dict(cuq_arg=0), D.E_UNSUPPORTED), (dict(o_arg=0), D.E_DESC),
    (dict(v_arg=9), D.E_DESC), (dict(q_tokens=1 << 40), D.E_DESC)])
def test_packed_attention_refusals(fields, code):
    assert _code(_with(B.attention_packed(10, 3, 8, 2), "pattn", **fields)) == code


def test_row_strides_whose_product_passes_64_bits_are_refused():
    n, row = (1 << 27) + 1, 1 << 37                                  # the last row starts at 2^64
    assert _code(_with(B.attention_packed(10, 3, 8, 2), "pattn", q_tokens=n, q_row=row, o_row=row)) == D.E_OOB
    assert _code(_with(B.attention_packed(10, 3, 8, 2), "pattn", k_tokens=n, k_row=row, v_row=row)) == D.E_OOB
    for make in (B.kv4_store, B.kv4_load):
        assert _code(_with(make(shape(), 7), "kv4", tokens=n, a_row=row, b_row=row)) == D.E_OOB


@pytest.mark.parametrize("make", [lambda c: B.kv4_store(c, 7), lambda c: B.kv4_load(c, 7), lambda c: B.attention_kv4(c, 6)])
@pytest.mark.parametrize("fields,code", [
    (dict(dim=32), D.E_UNSUPPORTED), (dict(group=16), D.E_UNSUPPORTED), (dict(page_size=8), D.E_UNSUPPORTED),
    (dict(page_size=24), D.E_UNSUPPORTED), (dict(pages=10), D.E_OOB), (dict(layers=3), D.E_OOB), (dict(layer=2), D.E_DESC),
    (dict(layer=-1), D.E_DESC), (dict(slots=4), D.E_OOB), (dict(slots=D.KV4_SLOTS + 1), D.E_UNSUPPORTED),
    (dict(max_pages=5), D.E_OOB), (dict(max_pages=1 << 40), D.E_DESC), (dict(hkv=0), D.E_DESC), (dict(a_off=1), D.E_UNSUPPORTED),
    (dict(a_off=1 << 20), D.E_OOB), (dict(b_row=12), D.E_UNSUPPORTED), (dict(pool_arg=-1), D.E_DESC), (dict(lens_arg=99), D.E_DESC)])
def test_cache_refusals(make, fields, code):
    assert _code(_with(make(shape()), "kv4", **fields)) == code


def test_cache_refusals_of_types():
    d = B.attention_kv4(shape(), 6)
    d.arg_dtype[0] = D.DTYPE_CODE["float32"]
    assert _code(d) == D.E_UNSUPPORTED
    d = B.attention_kv4(shape(), 6)
    d.arg_dtype[d.p.kv4.b_arg] = D.DTYPE_CODE["float16"]      # q and o of two types
    assert _code(d) == D.E_UNSUPPORTED
    assert _code(_with(B.attention_kv4(shape(), 6), "kv4", hq=5)) == D.E_DESC
    assert _code(_with(B.attention_kv4(shape(), 6), "kv4", scale=-1.0)) == D.E_UNSUPPORTED
    d = B.kv4_store(shape(), 7)
    d.units = 2
    assert _code(d) == D.E_DESC
    for bad in (dict(dim=96), dict(page_size=48), dict(group=128, dim=64)):
        with pytest.raises(ValueError):
            B.kv4_cache(slots=1, max_pages=1, pages=1, hkv=1, **bad)


@pytest.mark.parametrize("make,fields,code", [
    (lambda c: B.pages_grow(c, 2), dict(op=9), D.E_DESC), (lambda c: B.pages_grow(c, 2), dict(n=3), D.E_OOB),
    (lambda c: B.pages_grow(c, 2), dict(n=D.PAGES_IDS + 1), D.E_UNSUPPORTED), (lambda c: B.pages_grow(c, 2), dict(n=-1), D.E_DESC),
    (lambda c: B.pages_grow(c, 2), dict(pages=10), D.E_OOB), (lambda c: B.pages_grow(c, 2), dict(slots=0, n=2), D.E_DESC),
    (lambda c: B.pages_grow(c, 2), dict(page_size=0), D.E_DESC), (lambda c: B.pages_grow(c, 2), dict(pages=0), D.E_DESC), (lambda c: B.pages_grow(c, 2), dict(aux_arg=-1), D.E_DESC),
    (lambda c: B.pages_fork(c, 2), dict(pool_arg=-1), D.E_DESC), (lambda c: B.pages_fork(c, 2), dict(layers=3), D.E_OOB),
    (lambda c: B.pages_fork(c, 2), dict(page_bytes=24), D.E_DESC), (lambda c: B.pages_free(c, 2), dict(max_pages=5), D.E_OOB),
    (lambda c: B.pages_compact(c), dict(n=1), D.E_DESC), (lambda c: B.pages_compact(c), dict(pool_arg=0), D.E_UNSUPPORTED)])
def test_page_refusals(make, fields, code):
    assert _code(_with(make(shape()), "pages", **fields)) == code


@pytest.mark.parametrize("slots", [1, 64, 464, 465, 600, 1024, 4096])
@pytest.mark.parametrize("dim,group,per", [(128, 64, 4), (128, 128, 8), (128, 32, 4), (64, 64, 3), (64, 32, 12)])
def test_cache_attention_cuts_its_work_for_the_warps_an_sm_holds(slots, dim, group, per):
    """The workspace has two parts a warp, for as many CTAs of four warps as fit the 228 KB of an SM's shared memory: a tile ring of two
    stages a warp, 12 bytes a stage, 6 bytes a slot, 1 KB that the hardware keeps."""
    c = shape(dim=dim, group=group, hkv=1, slots=slots)
    floats = native.workspace_size(D.to_bytes(B.attention_kv4(c, per))) // 4 - slots - 1
    ctas, rest = divmod(floats, 2 * 4 * 148 * 16 * (dim + 2))
    smem = 8 * (64 * (dim + 8 * (dim // group)) + 12) + 32 + 6 * (slots + 1) + 1024
    assert rest == 0 and 2 <= ctas <= 3 and ctas * smem <= 228 * 1024


def halted_builders():
    c = shape()
    return [B.kv4_store(c, 7, halt=True), B.kv4_store(c, 7, fused_hq=4, halt=True), B.pages_grow(c, 2, halt=True), B.pages_fork(c, 2, halt=True),
            B.pages_fork(c, 2, deep=True, halt=True), B.pages_free(c, 2, halt=True), B.pages_compact(c, halt=True)]


@pytest.mark.parametrize("i", range(7))
def test_a_halt_word_is_the_last_argument(i):
    desc, names = halted_builders()[i], [f"a{k}" for k in range(16)]
    native.check(D.to_bytes(desc))
    last = desc.nargs - 1
    p, which = (desc.p.pages, "pages") if desc.kind == D.PAGES else (desc.p.kv4, "kv4")
    assert p.halt_arg_p1 == desc.nargs and desc.arg_numel[last] == 1
    sets = desc.kind == D.PAGES and p.op in (D.PAGES_OP["grow"], D.PAGES_OP["fork"], D.PAGES_OP["copy"])
    assert (last in RC.written_args(desc)) == sets
    streams = dma_access.streams(desc, 0, 1, names)
    assert {s["arg"] for s in streams} == set(names[:desc.nargs])
    assert {s["arg"] for s in streams if s["dir"] == "write"} == {names[k] for k in RC.written_args(desc)}
    assert _code(_with(desc, which, halt_arg_p1=desc.nargs + 1)) == D.E_DESC
    assert _code(_with(desc, which, halt_arg_p1=-1)) == D.E_DESC
    desc = halted_builders()[i]
    desc.arg_dtype[last] = D.DTYPE_CODE["int64"]
    assert _code(desc) == D.E_UNSUPPORTED
    desc = halted_builders()[i]
    desc.arg_numel[last] = 0
    assert _code(desc) == D.E_OOB


def test_reading_launches_take_no_halt_word():
    for desc in (B.kv4_load(shape(), 7), B.attention_kv4(shape(), 6)):
        assert _code(_with(desc, "kv4", halt_arg_p1=2)) == D.E_DESC


def test_launches_refuse_a_small_workspace_and_null_pointers_before_any_gpu():
    assert native.workspace_size(D.to_bytes(B.attention_kv4(shape(), 6))) > 0
    assert native.workspace_size(D.to_bytes(B.pages_fork(shape(), 2))) == 4 * (4 + 3 * 9)
    assert native.workspace_size(D.to_bytes(B.pages_free(shape(), 2))) == 0
    blob = D.to_bytes(B.pages_compact(shape()))
    with pytest.raises(native.ExecutorError) as e:
        native.launch(blob, [0, 1, 1, 1], 0, 1)
    assert e.value.code == D.E_ARGS


def test_builders_refuse_a_fused_projection_with_another_layout():
    for make in (lambda: B.attention_packed(8, 1, 4, 2, fused=True, head_major=True),
                 lambda: B.attention_packed(8, 1, 4, 2, fused=True, k_tokens=9),
                 lambda: B.kv4_store(shape(), 7, fused_hq=4, head_major=True)):
        with pytest.raises(ValueError):
            make()


class FakeCuda:
    """What workspace_for asks of torch: the current stream, which streams are being captured, and memory by stream."""

    def __init__(self):
        self.cuda, self.uint8, self.now, self.captured, self.taken = self, torch.uint8, self.stream_of(1), set(), []

    @staticmethod
    def stream_of(n):
        return types.SimpleNamespace(cuda_stream=n)

    def current_stream(self, device=None):
        return self.now

    @contextlib.contextmanager
    def stream(self, s):
        held, self.now = self.now, s
        yield
        self.now = held

    def is_current_stream_capturing(self):
        return self.now.cuda_stream in self.captured

    def empty(self, n, dtype, device):
        self.taken.append(self.now.cuda_stream)
        return torch.empty(n, dtype=dtype)


def test_a_workspace_comes_from_the_stream_its_launch_runs_on(monkeypatch):
    fake, device = FakeCuda(), torch.device("cuda", 0)
    monkeypatch.setattr(RC, "_torch", lambda: fake)
    monkeypatch.setattr(RC, "_workspaces", {})
    blob = D.to_bytes(B.attention_kv4(shape(), 6))
    own, side, third = RC.workspace_for(blob, device), fake.stream_of(2), fake.stream_of(3)
    assert fake.taken == [1] and RC.workspace_for(blob, device) is own
    other = RC.workspace_for(blob, device, side)
    assert fake.taken == [1, 2] and other is not own and RC.workspace_for(blob, device, side) is other
    fake.captured = {2, 3}                       # two branches of a capture, neither of them current
    for branch in (side, third):
        got = RC.workspace_for(blob, device, branch)
        assert got is not own and got is not other and fake.taken[-1] == branch.cuda_stream
    assert fake.now.cuda_stream == 1 and RC.workspace_for(blob, device) is own


def test_graph_binds_device_tensors_only():
    g = Graph("cuda:0")
    with pytest.raises(ValueError):
        g.bind("x", torch.zeros(4))


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on cuda:0 (what the launch boundary looks at; nothing is launched)."""
    is_cuda = True

    @property
    def device(self):
        return torch.device("cuda", 0)


def on_device(*shape, dtype):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def test_a_bound_buffer_keeps_its_size_and_type():
    g, t = Graph("cuda:0"), on_device(8, dtype=torch.int32)
    g.bind("x", t)
    g.bind("x", t)
    for other in (t[:4], t.view(torch.float32), on_device(8, dtype=torch.int32)):
        with pytest.raises(ValueError):
            g.bind("x", other)
    assert g.buffers["x"] is t


@pytest.mark.parametrize("current", [0, 1])
def test_a_graph_runs_and_synchronises_on_its_own_device(current, monkeypatch):
    class Cuda:
        now = current

        def current_device(self):
            return self.now

        @contextlib.contextmanager
        def device(self, d):
            held, self.now = self.now, d
            yield
            self.now = held

        def current_stream(self, device):
            return types.SimpleNamespace(cuda_stream=7)

    g, cuda, seen = Graph("cuda:0"), Cuda(), []
    g.torch = types.SimpleNamespace(cuda=cuda)
    g.steps = ["a step"]
    monkeypatch.setattr(g, "_launch", lambda i, stream: seen.append(("launch", cuda.now, stream)))
    monkeypatch.setattr(native, "sync", lambda stream: seen.append(("sync", cuda.now, stream)))
    g.run(sync=True)
    assert seen == [("launch", 0, 7), ("sync", 0, 7)] and cuda.now == current


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16])
def test_tensors_of_another_element_size_are_refused(dtype):
    """int64 lengths, as torch makes them, are not the int32 ones a launch reads."""
    c = shape()
    desc = B.pages_free(c, 2)
    ts = [on_device(n, dtype=torch.int32) for n in (2, c.slots * c.max_pages, c.slots, c.pages)]
    ts[2] = on_device(c.slots, dtype=dtype)
    with pytest.raises(RC.CudaError, match="argument 2"):
        RC.launch_tensors(D.to_bytes(desc), ts)
    g = Graph("cuda:0")
    for n, t in zip(("ids", "table", "lens", "refs"), ts):
        g.bind(n, t)
    with pytest.raises(ValueError, match="lens"):
        g.add("free", D.to_bytes(desc), ["ids", "table", "lens", "refs"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantisation_is_within_its_step(dtype, group):
    x = (torch.randn(50, 128, generator=torch.Generator().manual_seed(1)) * 3 + 1).to(dtype)
    x[0] = 2.5                                       # constant: exact
    x[1, :] = torch.tensor([-60000.0, 60000.0]).to(dtype).repeat(64)   # a range no sum of two can hold in fp16
    code, scale, mn = S.quantise(x, group)
    back = S.dequantised(x, group)
    assert torch.equal(back[0], x[0].double())
    assert int(code.min()) >= 0 and int(code.max()) == 15
    # Rounding: half a step; the rounded scale moves code 15 by 15 half units in the last place of the scale, the clamp by no more.
    step = scale.double().repeat_interleave(group, -1)
    assert bool(((back - x.double()).abs() <= step * (0.5 + 15 * torch.finfo(dtype).eps / 2) * (1 + 1e-6) + 1e-30).all())


def test_a_group_with_a_non_finite_value_stands_for_nan():
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    x[0, 3], x[1, 70], x[2, 0] = float("nan"), float("inf"), -float("inf")
    bad = torch.isnan(S.dequantised(x, 64))
    assert bad[0, :64].all() and not bad[0, 64:].any() and bad[1, 64:].all() and not bad[1, :64].any() and bad[2, :64].all()


@pytest.mark.parametrize("dim,page,group,hkv", SHAPES)
def test_records_hold_what_was_written(dim, page, group, hkv):
    c = shape(dim, page, group, hkv, slots=1, max_pages=2, pages=3)
    cache = S.Cache(c, torch.zeros(c.pool_bytes, dtype=torch.uint8), [[2, 0]], [page + 3])
    assert cache.pool.shape[-1] * hkv == c.page_bytes
    gen = torch.Generator().manual_seed(dim + page)
    k, v = (torch.randn(page + 3, hkv, dim, generator=gen).to(torch.bfloat16) for _ in "kv")
    for t in range(page + 3):
        for h in range(hkv):
            cache.write(0, t, h, k[t, h], v[t, h], layer=1)
    for t in range(page + 3):
        for h in range(hkv):
            a, b = cache.read(0, t, h, layer=1)
            assert torch.equal(a, S.dequantised(k[t, h], group)) and torch.equal(b, S.dequantised(v[t, h], group))
    # Every byte of a full record belongs to one token, K or V, code or parameter.
    seen = set()
    for kk, vv, kp, vp in cache.where:
        seen |= {b for b, _ in kk} | {b for b, _ in vv} | {p + i for p in kp + vp for i in range(4)}
    assert seen == set(range(c.page_bytes // hkv))


def test_page_oracle_forks_frees_and_compacts():
    pool = torch.arange(2 * 8 * 4).view(2, 8, 4)
    p = S.Pages([[-1] * 3 for _ in range(3)], [0, 0, 0], [0] * 8, pool, 4)
    p.grow([0, 1], [9, 4])
    assert p.table == [[0, 1, 2], [3, -1, -1], [-1] * 3] and p.refs == [1, 1, 1, 1, 0, 0, 0, 0]
    p.fork([0], [2])
    assert p.table[2] == [0, 1, 4] and p.refs == [2, 2, 1, 1, 1, 0, 0, 0] and torch.equal(p.pool[:, 4], p.pool[:, 2])
    p.free([1, 0])
    assert p.table[:2] == [[-1] * 3] * 2 and p.refs == [1, 1, 0, 0, 1, 0, 0, 0]
    p.compact()
    assert p.table[2] == [0, 1, 2] and p.refs == [1, 1, 1, 0, 0, 0, 0, 0]


def test_the_command_line_names_the_serving_kinds(capsys):
    from pytorchsim_triton_compiler import cli
    cli.target()
    got = json.loads(capsys.readouterr().out)["serving"]
    assert got == ["attn_packed", "kv4_store", "kv4_load", "attn_kv4", "pages"] and D.kind_name(D.PAGES) == "pages" and D.kind_name(99) == 99
