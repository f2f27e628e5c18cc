"""GPU: what a request of a shared batch brings of its own, the rules its tokens are drawn under and the log-probabilities it
asks for, against their definitions in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LAST = 1.0 - 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from cie_amd.kernels import ops

    return ops


def definition(row, temperature, uniform, top_k=0, top_p=1.0, min_p=0.0) -> int:
    """The token of one float32 row, by the definition, in 64 bits."""
    row = np.asarray(row, dtype=np.float64)
    known = np.where(np.isnan(row), -np.inf, row)
    best = known.max()
    first = int(known.argmax())
    if not temperature > 0 or best == -np.inf:
        return first
    with np.errstate(invalid="ignore", over="ignore"):
        weight = np.where(known == best, 1.0, np.exp((known - best) / np.float64(temperature)))
    weight = np.where(known == -np.inf, 0.0, np.nan_to_num(weight, nan=0.0))
    order = np.lexsort((np.arange(len(row)), -known))
    if 0 < top_k < len(row):
        order = order[:top_k]
    if top_p < 1:
        share = np.cumsum(weight[order])
        kept = (share - weight[order]) < np.float64(top_p) * share[-1]
        kept[0] = True
        order = order[: int(kept.sum())]
    if min_p > 0:
        order = order[weight[order] >= min(1.0, np.float64(min_p))]
    chosen = np.sort(order)
    running = np.cumsum(weight[chosen])
    place = int(np.searchsorted(running, np.float64(uniform) * running[-1], side="right"))
    return int(chosen[min(place, int(np.searchsorted(running, running[-1])))])


def draw(ops, logits, temperature, uniform, top_k=None, top_p=None, min_p=None):
    wide = lambda values, dtype: None if values is None else torch.tensor(values, dtype=dtype).cuda()  # noqa: E731
    return ops.sample(logits, wide(temperature, torch.float32), wide(uniform, torch.float32), top_k=wide(top_k, torch.int32),
                      top_p=wide(top_p, torch.float32), min_p=wide(min_p, torch.float32)).tolist()


def expected(logits, temperature, uniform, top_k=None, top_p=None, min_p=None):
    f32 = lambda values, r, off: off if values is None else float(np.float32(values[r]))  # noqa: E731
    return [definition(row, f32(temperature, r, 0), f32(uniform, r, 0), 0 if top_k is None else top_k[r], f32(top_p, r, 1.0),
                       f32(min_p, r, 0.0)) for r, row in enumerate(logits.cpu().numpy())]


def check(ops, logits, *rules, **named):
    got, want = draw(ops, logits, *rules, **named), expected(logits, *rules, **named)
    assert got == want, [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b]


VOCABS = [1, 2, 63, 64, 65, 1000, 4099, 16383, 32001, 65536, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("spread", [0.02, 2.5, 40.0])
def test_draws_under_every_rule(ops, vocab, spread):
    g = torch.Generator().manual_seed(vocab + int(spread * 100))
    rows = 24
    logits = torch.randn((rows, vocab), generator=g) * spread
    logits[::3, : max(1, vocab // 50)] += 4 * spread
    pick = lambda values: [values[i] for i in torch.randint(len(values), (rows,), generator=g)]  # noqa: E731
    check(ops, logits.cuda(), pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.7]), pick([0.0, LAST, 0.25, 0.5, 0.77, 0.123456]),
          pick([0, 0, -3, 1, 2, 5, 40, 50, 1000, vocab - 1, vocab, vocab + 7]), pick([1.0, 1.0, 0.0, 1e-7, 0.3, 0.8, 0.9, 0.95, 0.999, 2.0]),
          pick([0.0, 0.0, -1.0, 0.02, 0.1, 0.9, 1.0, 3.0]))


@pytest.mark.parametrize("rules", ["k", "p", "m"])
def test_each_rule_alone_and_rows_that_lie_apart(ops, rules):
    g = torch.Generator().manual_seed(5)
    rows, vocab = 33, 50001
    wide = torch.randn((rows, vocab + 13), generator=g).cuda() * 3
    logits = wide[:, 5: 5 + vocab]
    uniform = torch.rand(rows, generator=g).tolist()
    check(ops, logits, [0.9] * rows, uniform, top_k=[1 + 37 * r for r in range(rows)] if rules == "k" else None,
          top_p=[r / rows for r in range(rows)] if rules == "p" else None, min_p=[10.0 ** (-r / 8) for r in range(rows)] if rules == "m" else None)


@pytest.mark.parametrize("vocab", [200, 9000, 151936])
def test_equal_logits_go_by_their_index(ops, vocab):
    """Rows of few different values: the cut lies among equal ones, of which the lower indices are kept."""
    g = torch.Generator().manual_seed(vocab)
    rows = 20
    logits = torch.randint(0, 3, (rows, vocab), generator=g).float()
    logits[1] = 0.0
    logits[2] = -0.0
    logits[2, ::2] = 0.0  # (equal: one zero)
    logits[3, :] = 7.25
    uniform = [0.0, 0.5, LAST, 0.75] * 5
    check(ops, logits.cuda(), [1.0] * rows, uniform, [0, 3, vocab // 2, 10] * 5, [0.5, 1.0, 0.25, 0.9, 0.9999] * 4, [0.0] * rows)
    check(ops, logits.cuda(), [1.0] * rows, uniform, None, [0.5, 0.75, 0.25, 0.125] * 5, [0.0, 0.2] * 10)


@pytest.mark.parametrize("vocab", [130, 40000])
def test_rows_with_nothing_in_masked_places(ops, vocab):
    rows = 12
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g)
    lowest = torch.finfo(torch.float32).min
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2] = lowest
    logits[3, 5:] = -math.inf
    logits[4, : vocab - 3] = lowest
    logits[5, ::2] = math.nan
    logits[6, 77] = math.inf
    logits[7, 77] = logits[7, 101] = math.inf
    logits[8, 1:] = -math.inf
    logits[9, :-1] = math.nan
    logits[10] = -math.inf
    logits[10, vocab - 1] = lowest
    logits[11] = math.nan
    logits[11, 3] = -math.inf
    for uniform in (0.0, 0.6, LAST):
        for rule in (dict(top_k=[5] * rows), dict(top_p=[0.7] * rows), dict(min_p=[0.3] * rows),
                     dict(top_k=[50] * rows, top_p=[0.9] * rows, min_p=[0.05] * rows), dict(top_k=[0] * rows)):
            check(ops, logits.cuda(), [1.0] * rows, [uniform] * rows, **rule)
    check(ops, logits.cuda(), [0.0] * rows, [0.5] * rows, top_k=[3] * rows)


def test_temperatures_at_the_ends(ops):
    g = torch.Generator().manual_seed(3)
    temperature = [1e-30, 1e-3, 1e4, 1e30, -1.0, math.nan, 1.0, 1e-44]
    logits = torch.randn((8, 30000), generator=g) * 4
    for u in (0.1, LAST):
        check(ops, logits.cuda(), temperature, [u] * 8, [0, 100, 0, 100, 5, 5, 1, 0], [0.9, 1.0, 0.9, 0.5, 0.5, 0.5, 0.5, 0.5])


def test_infinite_temperatures_weigh_all_the_same(ops):
    g = torch.Generator().manual_seed(11)
    logits = torch.randn((6, 9001), generator=g)
    logits[:, ::7] = -math.inf
    check(ops, logits.cuda(), [math.inf] * 6, [0.0, 0.25, 0.5, 0.75, 0.9, LAST], [0, 0, 0, 0, 9, 0], [1.0, 1.0, 0.5, 0.5, 0.5, 1.0],
          [1.0, 0.3, 1.0, 0.0, 1.0, 0.0])


def test_a_weight_next_to_the_border_is_found_in_64_bits(ops):
    """Every token of 151,936 may be drawn: numbers right below and above a running share name the tokens on its two sides."""
    g = torch.Generator().manual_seed(8)
    rows, vocab = 16, 151936
    logits = (torch.randn((1, vocab), generator=g) * 0.5).repeat(rows, 1)
    uniform = (torch.randint(1 << 24, (rows,), generator=g).float() / (1 << 24)).tolist()
    check(ops, logits.cuda(), [1.0] * rows, uniform, [0] * rows, [1.0] * rows)
    check(ops, logits.cuda(), [1.0] * rows, uniform, [0] * rows, [0.99] * rows)


def test_a_draw_depends_on_its_own_row_alone(ops):
    g = torch.Generator().manual_seed(9)
    rows, vocab = 70, 33001
    logits = (torch.randn((rows, vocab), generator=g) * 3).cuda()
    uniform = torch.rand(rows, generator=g).tolist()
    k, p, m = [10 + r for r in range(rows)], [0.5 + r / 200 for r in range(rows)], [0.01 * (r % 3) for r in range(rows)]
    together = draw(ops, logits, [0.8] * rows, uniform, k, p, m)
    for r in (0, 1, 35, 69):
        assert draw(ops, logits[r: r + 1], [0.8], uniform[r: r + 1], k[r: r + 1], p[r: r + 1], m[r: r + 1]) == together[r: r + 1]


def test_rules_off_agree_with_the_draw_without_rules(ops):
    """The draw without rules sums in float32: its share of [0, 1) and this one's differ by its rounding only, so with numbers
    in the middle of a token's share both name the token."""
    logits = torch.tensor([[0.0, 1.0, 2.0, -1.0]]).repeat(4, 1).cuda()
    share = torch.softmax(logits[0].double() / 0.8, 0).cumsum(0).tolist()
    middle = [(a + b) / 2 for a, b in zip([0.0] + share[:-1], share)]
    assert draw(ops, logits, [0.8] * 4, middle, [0] * 4) == draw(ops, logits, [0.8] * 4, middle) == [0, 1, 2, 3]


def logprob_bound(vocab, value):
    # at most ceil(vocab / 256) terms join one running sum, each with an exponential off by 2 units in the last place, a
    # rescaling (2 roundings and one exponential) and an addition; some 20 joins of sums; the logarithm and two subtractions
    return (8 * -(-vocab // 256) + 100) * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(value))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 255), (2, 256), (7, 1001), (1, 151936), (8, 151936), (64, 40001),
                                        (300, 5003), (1100, 1025)])
def test_token_logprobs(ops, rows, vocab):
    g = torch.Generator().manual_seed(rows + vocab)
    wide = torch.randn((rows, vocab + 3), generator=g) * torch.linspace(0.1, 30.0, rows)[:, None]
    for logits in (wide[:, :vocab].contiguous().cuda(), wide.cuda()[:, 1: vocab + 1]):
        tokens = torch.randint(vocab, (rows,), generator=g, dtype=torch.int32).cuda()
        got = ops.token_logprobs(logits, tokens)
        assert got.dtype == torch.float32 and tuple(got.shape) == (rows,)
        want = torch.log_softmax(logits.cpu().double(), 1).gather(1, tokens.cpu().long()[:, None])[:, 0]
        for r in range(rows):
            a, b = got[r].item(), want[r].item()
            assert abs(a - b) <= logprob_bound(vocab, b), (r, a, b)


@pytest.mark.parametrize("vocab", [6, 3001, 151936])
def test_token_logprobs_of_odd_rows(ops, vocab):
    logits = torch.zeros((9, vocab))
    logits[0] = -math.inf                      # nothing at all: NaN
    logits[1, 2:] = -math.inf                  # two tokens left
    logits[2, 3] = math.nan
    logits[3, 4] = math.inf
    logits[4] = torch.finfo(torch.float32).min  # equal, however low
    logits[5, :-1] = torch.finfo(torch.float32).min
    logits[6] = 1e4
    logits[7, 1] = -math.inf
    tokens = torch.tensor([0, 1, 0, 0, 5, vocab - 1, 0, 1, vocab], dtype=torch.int32)
    got = ops.token_logprobs(logits.cuda(), tokens.cuda()).tolist()
    assert all(math.isnan(got[r]) for r in (0, 2, 3, 8))
    bound = logprob_bound(vocab, math.log(vocab))
    assert abs(got[1] + math.log(2)) <= bound and got[7] == -math.inf
    assert abs(got[4] + math.log(vocab)) <= bound and abs(got[6] + math.log(vocab)) <= bound and got[5] == 0.0
    outside = torch.tensor([-1, -(1 << 31), (1 << 31) - 1], dtype=torch.int32).cuda()
    assert all(math.isnan(v) for v in ops.token_logprobs(logits[6:9].cuda(), outside).tolist())


def test_drawn_tokens_and_their_logprobs_in_a_replayed_graph(ops):
    """A run of both, as a step would capture it: every replay on new logits and numbers gives what the eager calls give."""
    g = torch.Generator().manual_seed(31)
    rows, vocab = 9, 40003
    logits = torch.randn((rows, vocab), generator=g).cuda() * 3
    temperature, uniform = torch.full((rows,), 0.9).cuda(), torch.rand(rows, generator=g).cuda()
    k = torch.tensor([0, 1, 5, 50, 1000, 0, 0, 20000, 40], dtype=torch.int32).cuda()
    p = torch.tensor([0.9, 1.0, 0.5, 0.95, 0.9, 1.0, 0.99, 0.99, 1.0]).cuda()
    m = torch.tensor([0.0, 0.0, 0.1, 0.0, 0.0, 0.05, 0.0, 0.0, 0.0]).cuda()

    def both():
        tokens = ops.sample(logits, temperature, uniform, top_k=k, top_p=p, min_p=m)
        return tokens, ops.token_logprobs(logits, tokens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, scores = both()
    for turn in range(4):
        logits.copy_(torch.randn((rows, vocab), generator=g) * (turn + 1))
        uniform.copy_(torch.rand(rows, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager_tokens, eager_scores = both()
        assert torch.equal(tokens, eager_tokens) and torch.equal(scores, eager_scores)
        assert tokens.tolist() == expected(logits, [0.9] * rows, uniform.tolist(), k.tolist(), p.tolist(), m.tolist())


def test_calls_on_two_streams_at_once(ops):
    g = torch.Generator().manual_seed(32)
    logits = [torch.randn((12, 60001), generator=g).cuda() * 2 for _ in range(2)]
    uniform = [torch.rand(12, generator=g).cuda() for _ in range(2)]
    temperature, p = torch.ones(12).cuda(), torch.full((12,), 0.9).cuda()
    alone = [ops.sample(l, temperature, u, top_p=p).tolist() for l, u in zip(logits, uniform)]
    scores = [ops.token_logprobs(l, torch.tensor(a, dtype=torch.int32).cuda()).tolist() for l, a in zip(logits, alone)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                tokens = ops.sample(logits[i], temperature, uniform[i], top_p=p)
                got[i].append((tokens, ops.token_logprobs(logits[i], tokens)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(t.tolist() == alone[i] and s.tolist() == scores[i] for t, s in got[i])


def test_no_rows(ops):
    empty = torch.empty((0, 77)).cuda()
    none = torch.empty(0).cuda()
    assert ops.sample(empty, none, none, top_p=none).shape == (0,)
    assert ops.token_logprobs(empty, none.int()).shape == (0,)


def test_refusals(ops):
    logits, rows = torch.zeros((3, 100)).cuda(), torch.zeros(3).cuda()
    k = torch.zeros(3, dtype=torch.int32).cuda()
    ops.sample(logits, rows, rows, top_k=k)
    bad = [
        dict(logits=logits.half()), dict(logits=logits.cpu()), dict(logits=logits.t()), dict(logits=logits[:, :0]),
        dict(logits=logits[:1].expand(3, 100)),
        dict(temperature=None), dict(uniform=None), dict(temperature=rows[:2]), dict(uniform=rows.double()),
        dict(top_k=k.long()), dict(top_k=k[:2]), dict(top_p=rows[:1]), dict(min_p=k), dict(top_p=rows.cpu()),
        dict(out=torch.zeros(3).cuda()), dict(out=k[:2]),
    ]
    for change in bad:
        given = dict(logits=logits, temperature=rows, uniform=rows, top_k=k)
        given.update(change)
        with pytest.raises(ValueError):
            ops.sample(**given)
    for change in (dict(logits=logits.half()), dict(logits=logits.cpu()), dict(tokens=k.long()), dict(tokens=k[:2]), dict(out=k),
                   dict(logits=logits.t())):
        given = dict(logits=logits, tokens=k)
        given.update(change)
        with pytest.raises(ValueError):
            ops.token_logprobs(**given)


def test_short_lists_of_many_rows_at_once(ops):
    """Rows that one wave finishes alone, several workgroups a unit, with work of another stream beside them: the number that the
    wave draws must not be taken for the list's length by a wave that comes late."""
    g = torch.Generator().manual_seed(41)
    rows, vocab = 1500, 9001
    logits = torch.randn((rows, vocab), generator=g) * 3
    uniform, k = torch.rand(rows, generator=g).tolist(), [1 + r % 50 for r in range(rows)]
    want = expected(logits, [1.0] * rows, uniform, k)
    assert sum(64 < token <= 4096 for token in want) > 300 and sum(token > 4096 for token in want) > 300
    on = logits.cuda(), torch.ones(rows).cuda(), torch.tensor(uniform).cuda(), torch.tensor(k, dtype=torch.int32).cuda()
    beside = torch.randn((4096, 4096), generator=g).cuda()
    torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    for _ in range(6):
        with torch.cuda.stream(side):
            beside = torch.sin(beside)
        got.append(ops.sample(*on[:3], top_k=on[3]))
    torch.cuda.synchronize()
    for tokens in got:
        assert tokens.tolist() == want


@pytest.mark.parametrize("rows,kinds", [(130, "kpm"), (256, "pm"), (256, "p"), (300, "m")])
def test_rows_of_which_a_workgroup_takes_several_parts(ops, rows, kinds):
    """So many rows that a launch has fewer workgroups for a row than the row has parts."""
    vocab = 151936
    assert ops.RULES_SPREAD // rows < -(-vocab // ops.RULES_PART)
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * torch.linspace(0.3, 4.0, rows, device="cuda")[:, None]
    logits[::4, 1000:1500] += 6.0
    h = torch.Generator().manual_seed(rows)
    pick = lambda values: [values[i] for i in torch.randint(len(values), (rows,), generator=h)]  # noqa: E731
    uniform = torch.rand(rows, generator=h).tolist()
    check(ops, logits, pick([0.0, 0.5, 1.0, 1.0, 1.5]), uniform, pick([0, 0, 0, 20, 100]) if "k" in kinds else None,
          pick([1.0, 0.2, 0.5, 0.9, 0.99, 0.9999]) if "p" in kinds else None, pick([0.0, 0.0, 1e-6, 0.01, 0.3]) if "m" in kinds else None)


@pytest.mark.parametrize("vocab", [262145, 1048579, 1100003, (1 << 22) - 1, 1 << 22])
def test_the_largest_vocabularies(ops, vocab):
    """More chunks than a row's threads read at once, more parts than a workgroup has threads, and the limit itself.  (Such rows'
    weights are whole numbers of 2^-40 at the least: none of these, 20 below the largest at most (2^-29), counts as nothing, and
    their roundings, up to 2^-41 each, add up to some 2^-30 of the largest weight, where a row's sum is thousands of it and a
    uniform number has 24 bits.)"""
    assert ops.MAX_RULE_VOCAB == 1 << 22
    g = torch.Generator().manual_seed(vocab)
    rows = 8
    logits = torch.randn((rows, vocab), generator=g).clamp_(-4.0, 4.0) * 1.5
    logits[1] *= 0.01
    logits[2, vocab - 70000:] += 8.0
    logits[3, vocab - 1] = 30.0
    logits[4, ::3] = -math.inf
    logits[5, : vocab // 2] = torch.finfo(torch.float32).min
    logits[6] = torch.randint(0, 3, (vocab,), generator=g).float()
    uniform = [0.1, 0.5, LAST, 0.3, 0.77, 0.9, 0.25, 0.6]
    check(ops, logits.cuda(), [1.0] * rows, uniform, [0, 0, 5000, 40, 0, 0, 1000, vocab - 1], [0.9, 0.5, 1.0, 0.9, 0.99, 1.0, 0.9, 0.7],
          [0.0, 0.0, 0.0, 0.1, 0.0, 0.01, 0.0, 0.0])
    check(ops, logits.cuda(), [1.0] * rows, uniform, [1, 50, 300, 0, 2000, 20, 0, 0], [1.0, 0.9, 1.0, 1.0, 1.0, 0.5, 0.5, 1.0])


def test_refusals_beyond_the_limits(ops):
    most_rows, most = ops.MAX_RULE_ROWS, ops.MAX_RULE_VOCAB
    for rows, vocab in ((1, most + 1), (most_rows + 1, 2)):
        logits, per_row = torch.zeros((rows, vocab)).cuda(), torch.zeros(rows).cuda()
        with pytest.raises(ValueError):
            ops.sample(logits, per_row, per_row, top_p=per_row)
    with pytest.raises(ValueError):
        ops.token_logprobs(logits, per_row.int())
    logits, per_row = torch.zeros((most_rows, 2)).cuda(), torch.ones(most_rows).cuda()
    logits[1::2, 1] = 2.0
    alternating = [0, 1] * (most_rows // 2) + [0]
    for rule in (dict(top_k=torch.ones(most_rows, dtype=torch.int32).cuda()), dict(top_p=per_row * 0.0), dict(min_p=per_row)):
        tokens = ops.sample(logits, per_row, per_row * 0.0, **rule)
        # (two equal logits: the lower index; one that is larger: that one)
        assert tokens.tolist() == alternating, list(rule)
    scores = ops.token_logprobs(logits, tokens).tolist()
    assert all(abs(score - want) < 1e-6 for score, want in zip(scores, [-math.log(2), -math.log1p(math.exp(-2))] * (most_rows // 2)))
