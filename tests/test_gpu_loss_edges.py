"""The choice losses where they can go wrong beside the plain sizes: offsets that
change under a call, very uneven items, infinite ratios and KL terms, sums that
must be exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def offsets(lengths, lead=0):
    return lead + np.concatenate([[0], np.cumsum(lengths)])


def test_offsets_that_change_under_the_call(dp):
    """The results of such a call are of no use, but it ends, keeps to its
    arrays, and the next one is right.  Both layouts hold the same rows: in one
    a block's items fit into its stage, in the other every third block's do not."""
    pairs, each = 20_000, 5
    even = np.full(2 * pairs, each)
    uneven = np.zeros(2 * pairs, int)
    uneven[::1600] = 1600 * each
    a, b = (torch.from_numpy(offsets(n)).cuda() for n in (even, uneven))
    rows = int(even.sum())
    score = torch.randn(rows, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    want = dp.preference_loss(score, item_begin=a, hess=True)
    begin, side = a.clone(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(40):
        with torch.cuda.stream(side):
            for layout in (b, a, b, a):
                begin.copy_(layout)
        for _ in range(4):
            dp.preference_loss(score, item_begin=begin, hess=True)
    torch.cuda.synchronize()
    begin.copy_(a)
    got = dp.preference_loss(score, item_begin=begin, hess=True)
    assert all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("rows,classes", [(700, 4), (700, 5), (700, 40), (700, 300), (700, 3000), (3, 140_001)])
def test_vectors_in_each_others_place(dp, rows, classes):
    """A vector that a row loss writes may be one that it reads."""
    gen = torch.Generator("cuda").manual_seed(classes)
    z = torch.randn(rows, classes, generator=gen, device="cuda")
    y = torch.randint(-1, classes, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    old, adv = (torch.randn(rows, generator=gen, device="cuda") for _ in range(2))
    want = dp.policy_loss(z, y, old, adv, weight=adv, grad=True)
    loss, logp, grad = adv.clone(), old.clone(), torch.empty_like(z)
    dp.check(dp.lib().dp_policy_loss(0, z.data_ptr(), rows, classes, classes, y.data_ptr(), logp.data_ptr(), None,
                                     loss.data_ptr(), loss.data_ptr(), 0.2, 0.2, 0.0, loss.data_ptr(),
                                     logp.data_ptr(), grad.data_ptr(), classes, None, 0,
                                     torch.cuda.current_stream().cuda_stream))
    assert torch.equal(loss, want.loss) and torch.equal(logp, want.log_prob) and torch.equal(grad, want.grad)


def formula_rows(z64, y, c):
    """Gradient and curvature of sum c * log p(y), the coefficient's size finite."""
    p = np.exp(z64 - z64.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    hit = np.zeros_like(p)
    hit[np.arange(len(y)), y] = 1.0
    return c[:, None] * (hit - p), np.abs(c)[:, None] * np.maximum(2 * p * (1 - p), 1e-16)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("classes", [4, 6, 40, 90, 1500, 20_011, 140_001])
def test_chosen_classes_that_are_masked_and_ratios_past_the_range(dp, dtype, classes):
    """Rows whose chosen class is masked (kinds 0 and 1), whose ratio or whose
    reference's lead passes fp32's range (2 and 3), and plain ones (4), with
    advantages of each sign and none."""
    rows = 30
    rng = np.random.default_rng(classes)
    y = rng.integers(0, classes, rows).astype(np.int32)
    kind, adv = np.arange(rows) % 5, np.tile(np.repeat([1.5, -2.0, 0.0], 5), 2).astype(np.float32)
    z = torch.from_numpy(rng.standard_normal((rows, classes)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    z64 = z.double().cpu().numpy()
    for r in range(rows):
        if kind[r] in (0, 1):
            z64[r, y[r]] = -np.inf
        if classes > 4:  # other masks beside the chosen class
            z64[r, (y[r] + 1) % classes] = -np.inf
    z.copy_(torch.from_numpy(z64).to(z.dtype))
    up = lambda v: torch.from_numpy(np.asarray(v, np.float32)).cuda()  # noqa: E731
    yd = torch.from_numpy(y).cuda()
    with np.errstate(divide="ignore"):
        logp64 = (z64 - z64.max(1, keepdims=True) - np.log(np.exp(z64 - z64.max(1, keepdims=True)).sum(1, keepdims=True)))
    logp64 = logp64[np.arange(rows), y]
    # p is off by the sum's and the exponential's error, below 2^-12 at this many
    # classes; a coefficient by log p's, below 1e-4; a gradient is rounded to its type
    step = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]

    def check(g, h, c):
        g, h = g.double().cpu().numpy(), h.double().cpu().numpy()
        want_g, want_h = formula_rows(z64, y, c)
        size = np.abs(c)[:, None]
        past = np.abs(want_g) > (65520 if dtype == "float16" else 3e38)
        assert not np.isnan(g).any() and not np.isnan(h).any()
        assert np.array_equal(g[past], np.sign(want_g[past]) * np.inf)
        off = np.abs(np.where(past, 0.0, g) - np.where(past, 0.0, want_g))
        assert np.all(off <= (step + 2.0 ** -12) * np.abs(want_g) + 1e-4 * size + 2.0 ** -24)
        assert np.all(np.abs(h - want_h) <= 2.0 ** -11 * want_h + 1e-4 * size + 1e-30)
        assert np.all(g[hidden] == 0)
    hidden = (z64 == -np.inf) & (np.arange(classes)[None] != y[:, None])

    def large(r, at, sign):
        """The finite slope of rows where the formula's is past the range, from the curvature's floor and largest entry."""
        _, unit = formula_rows(z64, y, np.ones(rows))
        top = unit.argmax(1)
        size = (r.hess.double().cpu().numpy()[np.arange(rows), top] / unit[np.arange(rows), top])[at]
        assert np.all((size >= 2.0 ** 120) & (size <= 2.0 ** 126 * 1.001))
        return sign * size

    logp, norm = dp.log_prob(z, yd)
    assert np.array_equal(logp.cpu().numpy() == -np.inf, (kind == 0) | (kind == 1))
    seen = np.isfinite(logp64)
    assert np.allclose(logp.cpu().numpy()[seen], logp64[seen], rtol=0, atol=2e-4)
    c = rng.standard_normal(rows)
    check(*dp.log_prob_grad(z, yd, norm, up(c), hess=True), np.float32(c).astype(np.float64))

    base = np.where(seen, logp64, -3.0)
    old, ref = base - np.where(kind == 2, 100.0, 0.1), base + np.where(kind == 3, 100.0, 0.2)
    call = lambda **kw: dp.policy_loss(z, yd, up(old), up(adv), weight=up(np.full(rows, 0.5)), clip=(0.2, 0.3),  # noqa: E731
                                       hess=True, **kw)
    free = call()
    ratio = np.where(seen, np.exp(np.minimum(np.where(seen, logp64, 0) - old, 99.0)), 0.0)
    s1, s2 = ratio * adv, np.clip(ratio, 0.8, 1.3) * adv
    loss, slope = -0.5 * np.minimum(s1, s2), 0.5 * np.where(s1 <= s2, -s1, 0.0)
    wild = (kind == 2) & (adv < 0)  # e^100 passes fp32's range
    got = free.loss.double().cpu().numpy()
    assert np.all(got[wild] == np.inf) and np.allclose(got[~wild], loss[~wild], rtol=1e-3, atol=1e-6)
    slope[wild] = large(free, wild, 1)
    # kl 0: the reference's log-probabilities, infinite lead or not, count for nothing
    for other in (call(ref_log_prob=up(ref)), call(ref_log_prob=up(np.full(rows, -np.inf)))):
        assert all(torch.equal(u, v) for u, v in zip(other, free))
    kl = call(ref_log_prob=up(ref), kl=0.1)
    far = (kind == 3) | ~seen
    got = kl.loss.double().cpu().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        d = np.where(far, 0.0, ref - np.where(seen, logp64, 0.0))
        over = 0.5 * 0.1 * (np.expm1(d) - d)
    tame = ~(far | wild)
    assert np.all(got[~tame] == np.inf) and np.allclose(got[tame], (loss + over)[tame], rtol=1e-3, atol=1e-6)
    lead = slope - 0.5 * 0.1 * np.expm1(d)
    lead[far], lead[wild] = large(kl, far, -1), large(kl, wild, 1)
    check(free.grad, free.hess, slope)
    check(kl.grad, kl.hess, lead)


def exact_items(items, lengths):
    """Scores whose sums are exact by trees and by chains of up to 4095 terms, and
    not by longer chains: 4097 in each row of the long items (whose lengths are
    powers of two), small integers in the others."""
    rng = np.random.default_rng(items)
    score = rng.integers(-2, 3, int(lengths.sum())).astype(np.float32)
    begin = offsets(lengths)
    for i in np.flatnonzero(lengths >= 1 << 13):
        score[begin[i]:begin[i + 1]] = 4097.0
    return score, begin


@pytest.mark.parametrize("use_ref", [False, True])
@pytest.mark.parametrize("pairs,short", [(100_000, 2), (20_000, 10), (40_000, 15), (3000, 150)])
def test_very_long_items_among_short_ones(dp, pairs, short, use_ref):
    """A call of short items has items of 2^13, 2^14 and 2^20 rows: their sums are as
    exact as those of a call of long items, in any kernel of short ones."""
    lengths = np.full(2 * pairs, short)
    lengths[[7, 2 * pairs // 3 | 1, 2 * pairs - 4]] = 1 << 13, 1 << 20, 1 << 14
    lengths[600:606] = 0, 700, 700, 0, 5000, 3  # and some in between
    lengths[::17] = 0
    score, begin = exact_items(pairs, lengths)
    refs = np.where(np.abs(score) > 4000, 0.0, -1.0).astype(np.float32) if use_ref else None
    gap = score.astype(np.float64) - (refs if use_ref else 0.0)
    run = np.concatenate([[0.0], np.cumsum(gap)])
    total = run[begin[1:]] - run[begin[:-1]]
    beta = float(np.float32(2.0 ** -31))
    x = beta * (total[0::2] - total[1::2])  # of size 2 for the longest item
    assert 1.9 < np.abs(x).max() < 2.1
    up = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    r = dp.preference_loss(up(score), ref_score=up(refs), item_begin=up(begin), beta=beta, hess=True)
    # sums and their difference are exact: x, softplus and the sigmoids are rounded a few times each
    e = 2.0 ** -24
    loss, down = np.logaddexp(0, -x), 1 / (1 + np.exp(x))
    assert np.all(np.abs(r.loss.double().cpu().numpy() - loss) <= 16 * e * loss + 4 * e * np.abs(x) + 4 * e)
    q = np.repeat(np.stack([-beta * down, beta * down], 1).reshape(-1), lengths)
    h = np.repeat(np.maximum(beta * beta * down * (1 - down), 1e-16).repeat(2), lengths)
    off = 16 * e + 4 * e * np.repeat(np.abs(x).repeat(2), lengths)
    assert np.all(np.abs(r.grad.double().cpu().numpy() - q) <= beta * off)
    assert np.all(np.abs(r.hess.double().cpu().numpy() - h) <= beta * beta * off + 1e-22)


def test_gradients_go_on_into_autograd_by_hand(dp):
    """Results are detached; a gradient handed to backward() reaches what the margins came from."""
    x = torch.randn(50, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    w = torch.zeros(8, 5, device="cuda", requires_grad=True)
    y = torch.arange(50, device="cuda", dtype=torch.int32) % 5
    z = x @ w
    logp, norm = dp.log_prob(z, y)
    grad, _ = dp.log_prob_grad(z, y, norm, torch.ones(50, device="cuda"))
    assert not logp.requires_grad and not grad.requires_grad
    z.backward(grad)
    p = torch.full((50, 5), 0.2, device="cuda")
    hit = torch.nn.functional.one_hot(y.long(), 5).float()
    assert (w.grad - x.T @ (hit - p)).abs().max() < 1e-4  # (fp32 sums of 50 terms of size 3)
    with pytest.raises(dp.DPError, match="grad must be a tensor"):
        dp.log_prob_grad(z, y, norm, torch.ones(50, device="cuda"), grad=False)


PIECE = 8192  # rows that a block of the whole-device form takes
LONG = 1 << 18


@pytest.mark.parametrize("use_ref,smoothing", [(False, 0.0), (True, 0.1)])
@pytest.mark.parametrize("begin,tail", [
    ([0, 8191, 300_000], 0), ([8192, 5 * 8192, 40 * 8192], 5), ([8193, 8192 * 17 + 1, 8192 * 38 - 1], 1),
    ([8191, 8191, 8191 + LONG], 0), ([3, 3 + LONG, 3 + LONG], 9),
    # pairs just below, at and past the length that is cut into pieces, and one that makes their average long
    ([100, 9000, 32_867, 32_867, 65_635, 70_000, 98_404, 500_000, 1_200_000], 3),
    # eight pairs, empty ones and single rows among them
    (list(np.cumsum([16_384, 0, 0, 1, 0, 1_000_003, 3, 8192, 24_576, 250_001, 16_385, 1, 0, 400_000, 400_001, 7, 2])), 0)])
def test_few_pairs_of_very_many_rows_lose_no_piece(dp, begin, tail, use_ref, smoothing):
    """Small integers whose sums are exact in any order: a piece that is left out, or
    counted twice, moves its pair's loss by twenty times the bound or more."""
    begin = np.array(begin)
    pairs, rows = len(begin) // 2, int(begin[-1]) + tail
    assert pairs <= 8 and rows // pairs >= LONG
    rng = np.random.default_rng(rows)
    gap = rng.integers(-2, 3, rows).astype(np.float32)
    cuts = np.union1d(np.arange(0, rows, PIECE), begin[begin < rows])
    empty = np.add.reduceat(gap, cuts) == 0  # (no piece of an item sums to nothing)
    gap[cuts[empty]] += 1
    pieces = np.add.reduceat(gap, cuts)
    assert np.all(pieces != 0)
    refs = rng.integers(-9, 10, rows).astype(np.float32) if use_ref else None
    score = gap + refs if use_ref else gap
    run = np.concatenate([[0.0], np.cumsum(gap.astype(np.float64))])
    total = run[begin[1:]] - run[begin[:-1]]
    beta, smooth = 2.0 ** -10, float(np.float32(smoothing))
    x = beta * (total[0::2] - total[1::2])
    w = (0.5 + rng.random(pairs)).astype(np.float32)
    if pairs > 4:
        w[4] = 0.0
    up = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    r = dp.preference_loss(up(score), ref_score=up(refs), item_begin=up(begin), weight=up(w), beta=beta,
                           smoothing=smooth, hess=True)
    e = 2.0 ** -24
    up_, down = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    loss = (1 - smooth) * np.logaddexp(0, -x) + smooth * np.logaddexp(0, x)
    slope, bend = smooth * up_ - (1 - smooth) * down, up_ * down
    # a dozen roundings of terms no larger than 1 + |x|
    bound = 16 * e * (1 + np.abs(x))
    # what a piece of the smallest sum moves a loss by at least
    assert beta * np.abs(pieces).min() * np.minimum(up_, down).min() * (1 - 2 * smooth) > 20 * bound.max()
    assert np.all(np.abs(r.loss.double().cpu().numpy() - w * loss) <= w * bound)
    lengths = np.diff(begin)
    rowwise = lambda a, b, out: np.concatenate([np.full(begin[0], out), np.repeat(np.stack([a, b], 1).reshape(-1), lengths),  # noqa: E731
                                                np.full(tail, out)])
    g, h = r.grad.double().cpu().numpy(), r.hess.double().cpu().numpy()
    assert np.all(np.abs(g - rowwise(w * beta * slope, -w * beta * slope, 0.0)) <= rowwise(beta * bound, beta * bound, 0.0))
    want = np.maximum(w * beta * beta * bend, 1e-16)
    assert np.all(np.abs(h - rowwise(want, want, 1e-16)) <= rowwise(beta * beta * bound, beta * beta * bound, 0.0) + 1e-22)
