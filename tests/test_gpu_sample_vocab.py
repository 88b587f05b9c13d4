"""``map_sample_dev`` against the rule in extended precision: whole numbers, so they are equal wherever the draw is not within
2^-36 of another outcome (weights are rounded to 2^-45 of the largest; 2^18 such roundings add up to 2^-36 at most)."""
import numpy as np
import pytest

import adam_b200 as A
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu
MAP = 40


def draw(gpu, logits, rules, u, offsets=None, pad=0):
    """Tokens for the rows of ``logits``; offsets: where the rows lie in the map."""
    R, V = logits.shape
    offs = np.arange(R) * V + pad if offsets is None else np.asarray(offsets)
    end = int(offs.max()) + V
    gpu.map_create_typed(MAP, A.DTYPE_F32, 1, end + 2 * R)
    data = np.zeros(end + 2 * R, np.float32)
    for r in range(R):
        data[offs[r]:offs[r] + V] = logits[r]
    data[end:end + R] = u
    data[end + R:] = -7
    gpu.scatter_contiguous(MAP, 0, data)
    rule = np.zeros(R, A.SAMPLE_RULE)
    for r in range(R):
        rule[r] = rules[r % len(rules)]
    hs = [gpu.upload_dev(a)[0] for a in (offs.astype(np.uint32), rule, (end + np.arange(R)).astype(np.uint32), (end + R + np.arange(R)).astype(np.uint32))]
    gpu.map_sample_dev(MAP, *hs, R, V)
    out = gpu.gather(MAP, np.arange(end + R, end + 2 * R, dtype=np.uint32)).view(np.float32)
    for h in hs:
        gpu.free_handle(h)
    return out.astype(np.int64), [tuple(rule[r].tolist()) for r in range(R)]


def check(gpu, logits, rules, u, **kw):
    got, used = draw(gpu, logits, rules, u, **kw)
    close = 0
    for r in range(len(logits)):
        want, margin = ko.sample(logits[r], *used[r], u[r])
        if margin < 2.0 ** -36:
            close += 1
            continue
        assert got[r] == want, (r, used[r], float(u[r]), got[r], want, margin)
    assert close <= len(logits) // 8
    assert gpu.device_error() == 0
    return got


RULES = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 200, 1.0, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (1.1, 5000, 0.99, 0.01),
         (0.05, 3, 0.999, 0.0), (5.0, 1, 1.0, 0.0), (2.0, 0, 0.3, 0.2), (float("inf"), 7, 1.0, 0.0), (-1.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (13, 31), (12, 100), (24, 1000), (12, 4097), (13, 32003), (5, 65537), (12, 262144), (1, 262144), (70, 20011),
                                        (2, 700001), (149, 300)])
def test_rules_and_sizes(gpu, rows, vocab):
    rng = np.random.default_rng(rows * 1000 + vocab)
    logits = (rng.standard_normal((rows, vocab)) * 2.5 + 14.0 * rng.random((rows, vocab)) ** max(1, vocab / 40)).astype(np.float32)
    check(gpu, logits, RULES, rng.random(rows).astype(np.float32), pad=rows % 3)


@pytest.mark.parametrize("kind", ["peaked", "flat", "steps"])
@pytest.mark.parametrize("pad", [0, 3])
def test_rows_too_long_to_keep(gpu, kind, pad):
    """A CTA's share does not fit its shared memory; both cuts one after the other, of little and of much, ties across the cut."""
    rows, vocab = 12, 700001
    rng = np.random.default_rng(len(kind) + pad)
    x = rng.standard_normal((rows, vocab)) * 2.5
    if kind == "peaked":
        x += 14.0 * rng.random((rows, vocab)) ** (vocab / 40)
    logits = (np.round(x * 4) / 4 if kind == "steps" else x).astype(np.float32)
    rules = [(1.1, 5000, 0.99, 0.01), (1.0, 20000, 0.9, 0.0), (3.0, 200000, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 0.9, 0.02), (2.0, 700000, 0.5, 0.0),
             (0.02, 3000, 0.999, 0.0), (1.0, 300, 0.9, 0.1), (1.0, 0, 0.01, 0.0), (50.0, 0, 0.999, 0.0), (0.9, 2500, 1.0, 0.0), (1.0, 0, 1.0, 0.3)]
    check(gpu, logits, rules, rng.random(rows).astype(np.float32), pad=pad)


def plausible(x, temperature, top_k, top_p, u, got):
    """Can ``got`` be drawn with weights right to 5e-10 of themselves and half a unit of 2^-45?  Sums of equal small weights share
    their rounding, so the borders of the nucleus and of the draw are known to ``off``, not better."""
    w = np.exp((x.astype(np.longdouble) - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")[:top_k or None]
    c = np.cumsum(w[order])
    off = 5e-10 * (c[-1] - c[0]) + len(x) * 2.0 ** -46
    least, most = (min(int(np.searchsorted(c, top_p * c[-1] + d)) + 1, len(c)) for d in (-off, off))
    kept = np.sort(order[:most])
    off = 2 * off + c[most - 1] - c[least - 1]
    cum = np.cumsum(w[kept])
    at = int(np.searchsorted(kept, got))
    return at < len(kept) and kept[at] == got and cum[at] - w[got] <= u * cum[-1] + off and cum[at] >= u * cum[-1] - off


@pytest.mark.parametrize("rows", [20, 5])                   # streamed; in shared memory
@pytest.mark.parametrize("top_k,temperature", [(0, 1.0), (3000, 0.5), (200000, 2.0)])
@pytest.mark.parametrize("depth", [20.10165, 20.125])
@pytest.mark.parametrize("pad", [0, 3])
def test_groups_of_equal_logits_far_below_the_largest(gpu, rows, top_k, temperature, depth, pad):
    """A nucleus that takes nearly all of the weight, and most of the vocabulary ``depth`` temperatures below one logit, where the
    counts of a row too long to keep end (at half a bin of 1/64 temperature, at a bin's edge): a logit or some on this side of
    it, many on the other."""
    vocab = 262144
    rng = np.random.default_rng(top_k + pad + rows)
    kinds = []
    for above, below, spread in [(1, vocab, 0), (1500, vocab, 0), (vocab // 2, vocab, 0), (600, 700, 0), (0, 200000, 0.02)]:
        x = np.full(vocab, -45.0)
        x[:below] = -depth - 0.005
        x[:above] = -depth + 0.005
        x[:below] += spread * (rng.random(min(below, vocab)) - 0.5)
        kinds.append(x)
    logits = np.stack([rng.permutation(kinds[r % len(kinds)]) for r in range(rows)])
    logits[np.arange(rows), rng.integers(0, vocab, rows)] = 0.0
    logits = (logits * temperature + 3.0).astype(np.float32)
    u = (1 - 6e-4 * rng.random(rows)).astype(np.float32)
    got, used = draw(gpu, logits, [(temperature, top_k, p, 0.0) for p in (0.9995, 0.9999, 1 - 2.0 ** -20)], u, pad=pad)
    for r in range(rows):
        assert plausible(logits[r], used[r][0], top_k, used[r][2], float(u[r]), got[r]), (r, used[r], float(u[r]), got[r])
    assert len(set(got.tolist())) > rows // 3 and gpu.device_error() == 0


def test_special_logits_of_rows_too_long_to_keep(gpu):
    rng = np.random.default_rng(8)
    rows, vocab = 12, 700001
    logits = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    logits[:, 5] = logits[:, 600000] = np.inf            # infinities share what there is
    logits[3:6] = np.where(rng.random((3, vocab)) < 0.999, -np.inf, logits[3:6])
    logits[3:6, 5] = logits[3:6, 600000] = 3.0
    logits[6:9, 5:600001:7] = np.nan
    logits[6:9, 5] = logits[6:9, 600000] = 1.0
    logits[9] = 3.0e38 * np.sign(logits[9])
    logits[9, ::2] = 0.0
    logits[10], logits[11] = -np.inf, np.nan
    u = rng.random(rows).astype(np.float32)
    got, used = draw(gpu, logits, [(1.0, 0, 0.9, 0.0), (np.inf, 0, 0.9, 0.0), (0.7, 3000, 0.9, 0.01)], u)
    for r in (0, 1, 2):
        assert got[r] == (5 if u[r] < 0.5 else 600000), (r, u[r], got[r])
    for r in range(3, 10):
        x = logits[r].copy()
        x[np.isnan(x)] = -np.inf
        want, margin = ko.sample(x, *used[r], u[r])
        assert got[r] == want or margin < 2.0 ** -36, (r, used[r], u[r], got[r], want, margin)
    assert got[10] == got[11] == -1 and gpu.device_error() == 0


@pytest.mark.parametrize("vocab", [5, 3000, 50000, 262144])
def test_ties(gpu, vocab):
    """Few distinct logits: cuts fall inside groups of equal ones, of which the lowest indices stay."""
    rng = np.random.default_rng(vocab)
    rules = [(1.0, vocab // 2 + 1, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (0.9, vocab // 3 + 1, 0.77, 0.0), (1.0, 2, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.0, 0.0),
             (1.0, 0, 1.0, 1.0), (1.0, 0, -3.0, 7.0)]
    logits = rng.integers(0, 4, (8, vocab)).astype(np.float32)
    logits[:, ::7] *= -0.0                                   # both zeros are one logit
    check(gpu, logits, rules, rng.random(8).astype(np.float32))
    check(gpu, np.full((8, vocab), -1.25, np.float32), rules, rng.random(8).astype(np.float32))


def test_equal_halves_and_ends_of_the_unit_interval(gpu):
    """Sums of equal weights are exact, so their borders are too: a nucleus of exactly half, draws at 0 and just below 1."""
    logits = np.zeros((6, 8), np.float32)
    got, _ = draw(gpu, logits, [(1.0, 0, 0.5, 0.0), (1.0, 4, 1.0, 0.0)], np.array([0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.25, 0.25], np.float32))
    assert got.tolist() == [0, 0, 3, 3, 1, 1]


@pytest.mark.parametrize("vocab", [9, 5000, 262144])
def test_masked_and_special_logits(gpu, vocab):
    rng = np.random.default_rng(vocab + 1)
    low, inf, nan = np.float32(-3.402823466e38), np.float32(np.inf), np.float32(np.nan)
    base = rng.standard_normal(vocab).astype(np.float32)
    rows = []
    for fill in (-inf, nan, low):
        x = np.full(vocab, fill, np.float32)
        rows += [x.copy()]                                    # nothing, or nothing but the type's lowest
        x[vocab // 2], x[-1] = 1.0, 1.0
        rows += [x]
    x = base.copy()
    x[::3] = -inf
    x[1::3] = nan
    rows += [x]
    x = base.copy()
    x[[2, vocab - 2]] = inf                                    # two sure ones
    rows += [x]
    x = base.copy()
    x[4] = 3.4e38
    x[5] = low                                                # the difference overflows 32 bits
    rows += [x]
    rows = np.stack(rows)
    for rule in [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1e-30, 0, 0.5, 0.1), (1e30, 4, 0.9, 0.0)]:
        u = rng.random(len(rows)).astype(np.float32)
        got = check(gpu, rows, [rule], u)
        assert got[0] == got[2] == -1 and got[4] >= 0


def test_same_whatever_the_launch(gpu):
    """A row alone (many CTAs to it) and among others (few), twice each."""
    rng = np.random.default_rng(8)
    logits = (rng.standard_normal((150, 40000)) * 2).astype(np.float32)
    u = rng.random(150).astype(np.float32)
    many, _ = draw(gpu, logits, RULES, u)
    assert np.array_equal(many, draw(gpu, logits, RULES, u)[0])
    for r in range(0, 150, 13):
        assert draw(gpu, logits[r:r + 1], [RULES[r % len(RULES)]], u[r:r + 1])[0][0] == many[r]
    assert gpu.device_error() == 0


def test_bad_rules_and_offsets_are_left_out(gpu):
    logits = np.random.default_rng(2).standard_normal((5, 64)).astype(np.float32)
    nan = float("nan")
    rules = [(nan, 0, 1.0, 0.0), (1.0, 0, nan, 0.0), (1.0, 0, 1.0, nan), (1.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0)]
    got, _ = draw(gpu, logits, rules, np.array([0.5, 0.5, 0.5, 1.0, 0.5], np.float32))
    assert got[:4].tolist() == [-1] * 4 and got[4] >= 0
    assert gpu.device_error() == 8
    got, _ = draw(gpu, logits[:1], RULES, np.array([np.nan], np.float32))
    assert got[0] == -1 and gpu.device_error() == 8
    # a row that ends outside its map: the destination stays as it was
    gpu.map_create_typed(MAP, A.DTYPE_F32, 1, 100)
    gpu.scatter_contiguous(MAP, 0, np.full(100, 0.5, np.float32))
    hs = [gpu.upload_dev(np.array(v, np.uint32))[0] for v in ([40, 0], [90, 91], [95, 96])]
    rule = gpu.upload_dev(np.array([(1.0, 0, 1.0, 0.0)] * 2, A.SAMPLE_RULE))[0]
    gpu.map_sample_dev(MAP, hs[0], rule, hs[1], hs[2], 2, 64)
    assert gpu.gather(MAP, np.array([95, 96], np.uint32)).view(np.float32).tolist() == [0.5, 32.0]
    assert gpu.device_error() == 1


def test_refusals(gpu):
    gpu.map_create_typed(MAP, A.DTYPE_F32, 1, 100)
    gpu.map_create_typed(MAP + 1, A.DTYPE_F32, 2, 100)
    h, rule = gpu.upload_dev(np.zeros(2, np.uint32))[0], gpu.upload_dev(np.zeros(2, A.SAMPLE_RULE))[0]
    for args, code in [((MAP + 1, h, rule, h, h, 2, 8), -3), ((MAP, h, h, h, h, 2, 8), -4), ((MAP, h, rule, h, h, 3, 8), -4), ((MAP, 60000, rule, h, h, 2, 8), -4),
                       ((MAP, h, rule, h, h, 2, 0), -3), ((MAP, h, rule, h, h, 2, (1 << 24) + 1), -3), ((255, h, rule, h, h, 2, 8), -4)]:
        with pytest.raises(RuntimeError, match=f"code {code}"):
            gpu.map_sample_dev(*args)
    gpu.map_sample_dev(MAP, h, rule, h, h, 0, 8)
    gpu.map_destroy(MAP + 1)


def test_captured_draws_read_the_numbers_of_their_replay(gpu):
    rng = np.random.default_rng(5)
    V = 5000
    logits = rng.standard_normal((2, V)).astype(np.float32)
    gpu.map_create_typed(MAP, A.DTYPE_F32, 1, 2 * V + 4)
    hs = [gpu.upload_dev(np.array(v, np.uint32))[0] for v in ([0, V], [2 * V, 2 * V + 1], [2 * V + 2, 2 * V + 3])]
    rule = gpu.upload_dev(np.array([(1.0, 0, 1.0, 0.0)] * 2, A.SAMPLE_RULE))[0]
    graphs = []
    for _ in range(2):
        gpu.capture_begin()
        gpu.map_sample_dev(MAP, hs[0], rule, hs[1], hs[2], 2, V)
        graphs.append(gpu.capture_end())
    for i in range(4):
        u = rng.random(2).astype(np.float32)
        gpu.upload_dev(np.array([(1.0, 7 * i, 1.0, 0.0)] * 2, A.SAMPLE_RULE), rule)
        gpu.scatter_contiguous(MAP, 0, np.concatenate([logits.reshape(-1), u]))
        gpu.graph_launch(graphs[i % 2])
        got = gpu.gather(MAP, np.array([2 * V + 2, 2 * V + 3], np.uint32)).view(np.float32)
        assert got.tolist() == [ko.sample(logits[r], 1.0, 7 * i, 1.0, 0.0, u[r])[0] for r in range(2)]
    for g in graphs:
        gpu.graph_destroy(g)
