"""GPU: low-rank adapters of many requests beside a shared projection, against their definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cie_amd.kernels import ops

    return ops


def site(rows, k, columns, rank, count, dtype, stream=False, seed=0, adapters=None):
    """x, down, up, scale, adapters, into on the CPU, with odd values everywhere."""
    g = torch.Generator().manual_seed(seed)
    n, parts = sum(columns), len(columns)
    if adapters is None:
        adapters = torch.randint(-1, count, (rows,), generator=g)
    return dict(
        x=torch.randn((rows, k), generator=g).to(dtype), down=(torch.randn((count, parts * rank, k), generator=g) * k ** -0.5).to(dtype),
        up=(torch.randn((count, n, rank), generator=g) * rank ** -0.5).to(dtype), scale=torch.rand(count, generator=g) + 0.5,
        adapters=torch.as_tensor(adapters, dtype=torch.int32),
        into=torch.randn((rows, n), generator=g).to(torch.float32 if stream else dtype), columns=tuple(columns))


def definition(s):
    """The result in 64 bits, and how far a right kernel may be from it.

    A sum of n products in float32, in any order, is off by at most n 2^-24 of the sum of their sizes; the inner products may
    be held as two bfloat16 numbers (2^-17 of their size) on their way into the second one; then the scale, the addition and
    the rounding to the result's type (half a step)."""
    x, down, up = s["x"].double(), s["down"].double(), s["up"].double()
    out, size = s["into"].double().clone(), torch.zeros(s["into"].shape, dtype=torch.float64)
    rank, k = up.shape[2], x.shape[1]
    for a in range(down.shape[0]):
        rows = (s["adapters"] == a).nonzero()[:, 0]
        inner, inner_size = x[rows] @ down[a].t(), x[rows].abs() @ down[a].abs().t()
        begin = 0
        for part, width in enumerate(s["columns"]):
            mine, factor = slice(part * rank, (part + 1) * rank), up[a, begin: begin + width]
            out[rows, begin: begin + width] += float(s["scale"][a]) * (inner[:, mine] @ factor.t())
            size[rows, begin: begin + width] = float(s["scale"][a]) * (inner_size[:, mine] @ factor.abs().t())
            begin += width
    half_step = torch.finfo(s["into"].dtype).eps / 2
    bound = size * ((k + rank + 8) * 2.0 ** -24 + 2.0 ** -17) + out.abs() * (half_step + 2.0 ** -23)
    return out, bound * (1 + half_step)


def run(ops, s, out=None, **views):
    on = {name: value.cuda() if torch.is_tensor(value) else value for name, value in s.items()}
    on.update(views)
    return ops.lora_add(on["x"], on["down"], on["up"], on["scale"], on["adapters"], on["into"], columns=on["columns"], out=out)


def check(ops, s):
    want, bound = definition(s)
    got = run(ops, s).cpu().double()
    far = ((got - want).abs() > bound).nonzero()
    assert len(far) == 0, (len(far), far[:4].tolist(), [(got[tuple(i)].item(), want[tuple(i)].item(), bound[tuple(i)].item()) for i in far[:4]])
    none = s["adapters"] < 0
    assert torch.equal(got[none].to(s["into"].dtype), s["into"][none])  # (rows without an adapter: bit by bit)


KINDS = [("bfloat16", False), ("bfloat16", True), ("float32", False)]


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("rank,columns", [(16, (192, 64, 64)), (8, (200,)), (64, (320, 320)), (12, (36, 20))])
def test_rows_ranks_and_pieces(ops, dtype, stream, rows, rank, columns):
    check(ops, site(rows, 256, columns, rank, 5, getattr(torch, dtype), stream, seed=rows + rank))


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("rank", [1, 2, 3, 4, 5, 7, 24, 32, 40, 100, 128])
def test_ranks(ops, dtype, stream, rank):
    check(ops, site(37, 136, (80, 48), rank, 3, getattr(torch, dtype), stream, seed=rank))


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("k", [1, 7, 8, 30, 31, 32, 33, 64, 104, 520, 1000, 4864, 18944])
def test_lengths_of_a_row(ops, dtype, stream, k):
    check(ops, site(19, k, (72, 24), 8, 3, getattr(torch, dtype), stream, seed=k))


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("columns", [(1,), (3, 5), (17, 1, 30), (63, 65, 2, 126), (1000, 24), (15, 16, 17, 18)])
def test_odd_columns(ops, dtype, stream, columns):
    for rows in (3, 70):
        check(ops, site(rows, 96, columns, 16, 4, getattr(torch, dtype), stream, seed=len(columns)))


@pytest.mark.parametrize("dtype,stream", KINDS)
def test_numbers_of_many_adapters(ops, dtype, stream):
    """Numbers that differ in a single bit, low or high, beside rows without any."""
    bits = [1 << b for b in range(10)]
    adapters = [0, *bits, -1, 1023, *[1023 - b for b in bits], 0, 512, 513, *range(300, 340), -1, 1000, 1000, 512]
    for rows in (len(adapters), 16, 3):
        check(ops, site(rows, 64, (40,), 4, 1024, getattr(torch, dtype), stream, seed=rows, adapters=adapters[-rows:]))
    check(ops, site(4000, 64, (2048, 2048), 4, 1024, getattr(torch, dtype), stream, seed=9, adapters=(adapters * 60)[:4000]))


@pytest.mark.parametrize("dtype,stream", KINDS)
def test_who_has_which_adapter(ops, dtype, stream):
    """None at all, one for all, every row another one, runs that end inside a tile, numbers that name no adapter."""
    for seed, adapters in enumerate([
            [-1] * 70, [2] * 70, [r % 64 for r in range(140)], [r % 3 for r in range(200)], [0] * 63 + [1] * 2 + [3] * 64 + [-1] * 9,
            [-1] * 40 + [5] + [-1] * 40, [-(1 << 31), -2, 64, (1 << 31) - 1, 1, 63]]):
        s = site(len(adapters), 104, (48, 32), 16, 64, getattr(torch, dtype), stream, seed=seed, adapters=adapters)
        check(ops, s)
        if max(adapters) >= 64:  # (not an adapter: its row stays as it is)
            got = run(ops, s).cpu()
            assert torch.equal(got[:4], s["into"][:4])


@pytest.mark.parametrize("dtype,stream", KINDS)
def test_rows_that_lie_apart(ops, dtype, stream):
    dtype = getattr(torch, dtype)
    for k, shift in ((128, 8), (128, 1), (100, 3)):
        s = site(50, k, (96, 40), 16, 3, dtype, stream, seed=k + shift)
        want, bound = definition(s)
        x = torch.full((50, k + 24), math.nan, dtype=dtype).cuda()
        x[:, shift: shift + k] = s["x"].cuda()
        into = torch.full((50, 136 + 16), 5.0, dtype=s["into"].dtype).cuda()
        into[:, shift: shift + 136] = s["into"].cuda()
        out = torch.full((50, 136 + 32), 7.0, dtype=s["into"].dtype).cuda()
        run(ops, s, out=out[:, shift: shift + 136], x=x[:, shift: shift + k], into=into[:, shift: shift + 136])
        assert ((out[:, shift: shift + 136].cpu().double() - want).abs() <= bound).all()
        assert (out[:, :shift] == 7).all() and (out[:, shift + 136:] == 7).all() and (into[:, :shift] == 5).all()
        run(ops, s, x=x[:, shift: shift + k], into=into[:, shift: shift + 136])  # in place
        assert torch.equal(into[:, shift: shift + 136], out[:, shift: shift + 136])
        assert (into[:, :shift] == 5).all() and (into[:, shift + 136:] == 5).all()


@pytest.mark.parametrize("dtype,stream", KINDS)
def test_a_row_depends_on_its_own_adapter_alone(ops, dtype, stream):
    """Bit by bit the same alone, among others, and beside adapters and rows of infinities and NaN."""
    s = site(90, 264, (112, 48), 16, 6, getattr(torch, dtype), stream, seed=4)
    together = run(ops, s).cpu()
    for r in (0, 1, 17, 64, 89):
        one = {name: value[r: r + 1] if name in ("x", "adapters", "into") else value for name, value in s.items()}
        assert torch.equal(run(ops, one).cpu()[0], together[r]), r
    odd = {name: value.clone() if torch.is_tensor(value) else value for name, value in s.items()}
    odd["down"][2], odd["up"][2] = math.inf, math.nan
    odd["x"][s["adapters"] == 2] = math.nan
    odd["x"][s["adapters"] < 0] = math.inf
    got = run(ops, odd).cpu()
    others = s["adapters"] != 2
    assert torch.equal(got[others], together[others]) and not got[~others].isfinite().any()


def test_many_rows_and_columns(ops):
    """Offsets beyond a tile grid's first dimension, and a prompt whose rows take two adapters."""
    adapters = [0] * 900 + [2] * 700 + [-1] * 400 + [r % 4 for r in range(48)]
    check(ops, site(2048, 512, (4864, 4864), 32, 4, torch.bfloat16, seed=2, adapters=adapters))
    check(ops, site(1100, 3584, (2048,), 8, 3, torch.float32, seed=3))


@pytest.mark.parametrize("dtype,stream", KINDS)
def test_replayed_with_other_adapters(ops, dtype, stream):
    s = site(21, 256, (128, 64), 16, 4, getattr(torch, dtype), stream, seed=12)
    on = {name: value.cuda() if torch.is_tensor(value) else value for name, value in s.items()}
    call = lambda: ops.lora_add(on["x"], on["down"], on["up"], on["scale"], on["adapters"], on["into"],  # noqa: E731
                                columns=on["columns"], out=torch.empty_like(on["into"]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # (two graphs, whose workspaces must not be one)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call()))
        graphs[-1] = (graph, graphs[-1][1])
    g = torch.Generator().manual_seed(77)
    for _ in range(3):
        on["adapters"].copy_(torch.randint(-1, 4, (21,), generator=g).int())
        on["x"].copy_(torch.randn((21, 256), generator=g))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = call()
        assert all(torch.equal(out, eager) for _, out in graphs)
        now = dict(s, x=on["x"].cpu(), adapters=on["adapters"].cpu())
        want, bound = definition(now)
        assert ((eager.cpu().double() - want).abs() <= bound).all()


def test_no_rows(ops):
    s = site(0, 64, (32,), 8, 2, torch.bfloat16)
    assert run(ops, s).shape == (0, 32)


def test_refusals(ops):
    s = {name: value.cuda() if torch.is_tensor(value) else value for name, value in site(4, 64, (32, 16), 8, 2, torch.bfloat16).items()}
    ops.lora_add(**s)
    bad = [
        dict(x=s["x"].cpu()), dict(x=s["x"].half()), dict(x=s["x"].float()), dict(x=s["x"][:, :63]), dict(x=s["x"][0]),
        dict(x=s["x"][:1].expand(4, 64)), dict(x=s["x"].t()), dict(down=s["down"][:, :8].contiguous()), dict(down=s["down"][:, :, :32]),
        dict(down=s["down"][:1]), dict(up=s["up"][:, :, :4].contiguous()), dict(up=s["up"][:, :47].contiguous()), dict(up=s["up"].float()),
        dict(scale=s["scale"][:1]), dict(scale=s["scale"].double()), dict(adapters=s["adapters"].long()), dict(adapters=s["adapters"][:3]),
        dict(into=s["into"].half()), dict(into=s["into"][:3]), dict(into=s["into"][:, :47]), dict(columns=(32,)), dict(columns=(32, 17)),
        dict(columns=(32, 16, 0)), dict(columns=(48, 0)), dict(columns=None), dict(columns=(24, 8, 8, 4, 4)), dict(columns=()),
        dict(out=s["into"].float()), dict(out=s["into"][:3]), dict(out=s["into"].cpu()),
    ]
    for change in bad:
        with pytest.raises(ValueError):
            ops.lora_add(**dict(s, **change))
    wide = site(4, 64, (32,), 129, 2, torch.bfloat16)
    with pytest.raises(ValueError):
        run(ops, wide)
    wide = {name: value.cuda() if torch.is_tensor(value) else value for name, value in site(4, 64, (32,), 8, 2, torch.float32).items()}
    with pytest.raises(ValueError):
        ops.lora_add(**dict(wide, into=wide["into"].bfloat16()))


def test_more_columns_than_a_grids_second_dimension_has_blocks(ops):
    """Few rows of a rank that the form for many does not take; the widths end inside a block."""
    g = torch.Generator(device="cuda").manual_seed(6)
    columns = (8388480, 333, 70001)
    n, rank, k = sum(columns), 72, 8
    x = torch.randn((2, k), generator=g, device="cuda").bfloat16()
    down = torch.randn((2, 3 * rank, k), generator=g, device="cuda").bfloat16()
    up = torch.randn((2, n, rank), generator=g, device="cuda").bfloat16()
    scale, adapters = torch.tensor([0.5, 1.5], device="cuda"), torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    into = torch.randn((2, n), generator=g, device="cuda")
    got = ops.lora_add(x, down, up, scale, adapters, into, columns=columns, out=torch.empty_like(into))
    begin = 0
    for piece, width in enumerate(columns):
        for first in range(begin, begin + width, 1 << 20):
            part = slice(first, min(first + (1 << 20), begin + width))
            for row, a in enumerate((1, 0)):
                inner = down[a, piece * rank: (piece + 1) * rank].double() * x[row].double()
                factor = up[a, part].double()
                want = into[row, part].double() + scale[a].double() * (factor @ inner.sum(1))
                size = scale[a].double() * (factor.abs() @ inner.abs().sum(1))
                bound = size * ((k + rank + 8) * 2.0 ** -24 + 2.0 ** -17) + want.abs() * 2.0 ** -22  # (as definition() has it)
                assert ((got[row, part].double() - want).abs() <= bound).all(), (piece, first, row)
        begin += width


@pytest.mark.parametrize("rank", [3, 4, 8, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("rows,columns", [(1, 48), (37, 200), (2048, 4300)])
def test_the_streams_sums_keep_all_bits_of_32(ops, rows, columns, rank):
    """bfloat16 operands whose inner products are whole numbers of 24 bits times a power of two (three digits of 8 bits), each
    times a single 1 of `up`, into a float32 stream of zeros: every step is exact in 32 bits, so the result has to be equal."""
    g = torch.Generator().manual_seed(rows + rank)
    digits = torch.randint(128, 256, (2, rank, 3), generator=g) * (2 * torch.randint(0, 2, (2, rank, 1), generator=g) - 1)
    down = torch.zeros((2, rank, 24))
    down[:, :, [1, 10, 20]] = digits.float() * torch.tensor([65536.0, 256.0, 1.0])
    up = torch.nn.functional.one_hot(torch.randint(rank, (2, columns), generator=g), rank)
    x = torch.zeros((rows, 24))
    x[:, [1, 10, 20]] = 2.0 ** torch.randint(-8, 8, (rows, 1), generator=g)
    adapters = torch.randint(-1, 2, (rows,), generator=g)
    adapters[0] = 1
    s = dict(x=x.bfloat16(), down=down.bfloat16(), up=up.bfloat16(), scale=torch.tensor([1.0, 0.5]), adapters=adapters.int(),
             into=torch.zeros((rows, columns)), columns=(columns,))
    assert torch.equal(s["down"].float(), down)
    want = torch.zeros((rows, columns), dtype=torch.float64)
    for a in range(2):
        mine = adapters == a
        want[mine] = float(s["scale"][a]) * (x[mine].double() @ down[a].double().t()) @ up[a].double().t()
    assert torch.equal(want.float().double(), want)
    wrong = (run(ops, s).cpu() != want.float()).nonzero()
    assert len(wrong) == 0, (len(wrong), wrong[:4].tolist())


def plan_of(ops, s):
    """The plan that a call of these operands runs, and what it means."""
    (rows, k), (count, n, rank) = s["x"].shape, s["up"].shape
    share = 256 // s["x"].element_size()
    chunk, parts, tile_rows, _slots, block, up_slots = ops.plan_lora(rows, k, n, len(s["columns"]) * rank, rank, count, share, ops.compute_units())
    chunks = -(-k // chunk)
    return dict(parts="groups" if parts < chunks else "chunks" if parts > 1 else "one", tile_rows=tile_rows,
                up="strips" if up_slots == 0 else "rows", steps=-(-rank // (32 if s["x"].element_size() == 2 else 16)))


def runs_of(lengths, adapters, rows):
    """Rows in runs of these lengths, each with the next of these adapters."""
    out = []
    while len(out) < rows:
        out += [adapters[len(out) % len(adapters)]] * lengths[len(out) % len(lengths)]
    return out[:rows]


# rows, k, columns, rank, runs of rows with one adapter: prompts (whole tiles), some dozens of rows (two matrix tiles of an adapter), few
PROMPTS, DOZENS, FEW = [500, 64, 771], [20, 31, 33, 64], [1, 5, 3, 16, 2]
FORMS = [
    # 64-row tiles of the first product, K in chunks or in groups of them, one, two and four column tiles
    (4032, 4096, (192,), 16, PROMPTS, dict(parts="chunks", tile_rows=64)),
    (4032, 4096, (192,), 16, DOZENS, dict(parts="chunks", tile_rows=64)),
    (4100, 4096, (192,), 16, PROMPTS, dict(parts="groups", tile_rows=64)),
    (6000, 4104, (200,), 28, DOZENS, dict(parts="groups", tile_rows=64)),
    (2048, 1000, (96, 104), 64, PROMPTS, dict(parts="chunks", tile_rows=64, up="rows")),
    (2048, 1000, (96, 104), 64, FEW, dict(parts="chunks", tile_rows=64, up="rows")),
    (2111, 4096, (96, 104), 64, DOZENS, dict(parts="groups", tile_rows=64, up="rows")),
    (2111, 4096, (96, 104), 100, PROMPTS, dict(parts="groups", tile_rows=64, up="rows")),
    # the second product's form for many rows, at one, two and four steps of the rank, with whole strips alone, columns behind the last
    # one, pieces that do not begin on 16 bytes, tiles of one adapter and of many
    (2111, 4096, (2048, 2560), 64, PROMPTS, dict(parts="groups", tile_rows=64, up="strips")),
    (2111, 4096, (2100, 2504), 64, DOZENS, dict(parts="groups", tile_rows=64, up="strips")),
    (2111, 1000, (2048, 2560), 48, FEW, dict(up="strips")),
    (2111, 1000, (2101, 2555), 64, PROMPTS, dict(up="strips")),
    (2111, 1000, (2101, 2555), 36, FEW, dict(up="strips")),
    (2111, 520, (4664,), 44, DOZENS, dict(up="strips")),
    (2111, 520, (4664,), 20, PROMPTS, dict(up="strips")),
    (2111, 520, (4663,), 8, PROMPTS, dict(up="strips")),
]


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("rows,k,columns,rank,lengths,form", FORMS)
def test_forms_of_many_rows(ops, dtype, stream, rows, k, columns, rank, lengths, form):
    s = site(rows, k, columns, rank, 4, getattr(torch, dtype), stream, seed=rows + rank, adapters=runs_of(lengths, [2, 0, -1, 3, 1], rows))
    plan = plan_of(ops, s)
    if k > 1000 or dtype == "bfloat16":  # (chunks of float32 are half as long: other parts of a short K)
        assert {name: plan[name] for name in form} == form
    check(ops, s)
    beside = torch.full(s["into"].shape, 9.0, dtype=s["into"].dtype).cuda()
    assert torch.equal(run(ops, s, out=beside), run(ops, s))


def test_the_forms_of_many_rows_are_all_there(ops):
    seen = set()
    for dtype, stream in KINDS:
        for rows, k, columns, rank, _, _ in FORMS:
            shapes = dict(x=torch.empty((rows, k), dtype=getattr(torch, dtype), device="meta"), up=torch.empty((4, sum(columns), rank)), columns=columns)
            plan = plan_of(ops, shapes)
            seen |= {(dtype, plan["parts"], plan["tile_rows"]), (dtype, plan["up"], plan["steps"])}
    for dtype, steps in (("bfloat16", (1, 2)), ("float32", (1, 2, 3, 4))):
        assert {(dtype, "chunks", 64), (dtype, "groups", 64), *[(dtype, "strips", s) for s in steps]} <= seen, seen


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("rows,k,columns,rank", [(2300, 4096, (2100, 2504), 64), (2300, 4104, (2101, 2555), 20), (4200, 11008, (200,), 16),
                                                 (2300, 4096, (96, 104), 100)])
def test_a_row_is_the_same_in_every_form(ops, dtype, stream, rows, k, columns, rank):
    """Bit by bit: a prompt's rows in the forms for many rows, and the same rows alone or with some beside them."""
    s = site(rows, k, columns, rank, 4, getattr(torch, dtype), stream, seed=rank, adapters=runs_of(PROMPTS, [2, 0, -1, 3, 1], rows))
    together, plans = run(ops, s).cpu(), {str(plan_of(ops, s))}
    for first, count in ((0, 1), (63, 2), (rows - 1, 1), (490, 17), (560, 70), (700, 200), (30, 640), (900, 1300)):
        some = {name: value[first: first + count] if name in ("x", "adapters", "into") else value for name, value in s.items()}
        plans.add(str(plan_of(ops, some)))
        assert torch.equal(run(ops, some).cpu(), together[first: first + count]), (first, count, plan_of(ops, some), plan_of(ops, s))
    assert len(plans) > 1


def test_operands_that_the_matrix_cores_do_not_take_are_told_of(ops, monkeypatch):
    """Once for each kind: a rank, a length, a distance of the rows, a place; never where the tiles run."""
    import warnings

    def told(s, **views):
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            run(ops, s, **views)
        return [str(w.message) for w in seen if issubclass(w.category, RuntimeWarning) and "generic kernels" in str(w.message)]

    monkeypatch.setattr(ops, "_SAID_GENERIC", set())
    fine = site(5, 64, (32,), 8, 2, torch.bfloat16)
    wide = torch.zeros((5, 80), dtype=torch.bfloat16).cuda()
    apart = torch.zeros((5, 67), dtype=torch.bfloat16).cuda()
    assert told(fine) == [] and told(fine, x=wide[:, 8:72]) == []
    assert told(site(0, 60, (32,), 7, 2, torch.bfloat16)) == []
    cases = [(site(5, 64, (32,), 6, 2, torch.bfloat16), {}), (site(5, 60, (32,), 8, 2, torch.bfloat16), {}), (fine, dict(x=apart[:, :64])),
             (fine, dict(x=wide[:, 1:65]))]
    for s, views in cases:
        assert len(told(s, **views)) == 1 and told(s, **views) == []
    assert told(fine) == []
