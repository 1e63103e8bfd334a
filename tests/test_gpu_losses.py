"""The choice losses on the GPU against their formulas in 64 bits: at the sizes
where a kernel changes its way (classes in registers, in a block, past it), at
odd sizes, strides and alignments, and with masks that leave little or nothing."""
import numpy as np
import pytest

import loss_reference as ref64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = ["float32", "float16", "bfloat16"]
CLIP, KL = (0.2, 0.3), 0.05


def margins(rows, classes, dtype, seed, pad=0, shift=0, scale=2.0, offset=0.0):
    """Margins on the GPU, rows classes + pad apart, starting `shift` elements
    into their storage, and the same values in 64 bits."""
    rng = np.random.default_rng(seed)
    z = torch.from_numpy((rng.standard_normal((rows, classes)) * scale + offset).astype(np.float32))
    z = z.to(getattr(torch, dtype))
    store = torch.full((rows * (classes + pad) + shift,), float("nan"), dtype=z.dtype, device="cuda")
    view = store[shift:].view(rows, classes + pad)[:, :classes]
    view.copy_(z)
    return view, z.double().numpy(), rng


def labels(rng, rows, classes, ignored=0.2):
    y = rng.integers(0, classes, rows).astype(np.int32)
    miss = rng.random(rows)
    y[miss < ignored] = -1
    y[miss < ignored / 4] = classes  # past the classes is no label either
    return y


def near(got, want, bound, what):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, what
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what
    off = np.abs(got[~odd] - want[~odd])
    bound = np.broadcast_to(bound, want.shape)[~odd]
    worst = int(np.argmax(off - bound)) if off.size else 0
    assert not off.size or off[worst] <= bound[worst], (what, off[worst], bound[worst], want[~odd][worst])


def check_rows(dp, z, z64, y, rng, dtype, hess=True, in_place=False, weight=None):
    """log_prob, its gradient and the policy loss of one set of margins."""
    rows, classes = z64.shape
    yd = torch.from_numpy(y).cuda()
    logp, top, log_sum, p, live, none = ref64.softmax_rows(z64, y)
    dl = ref64.log_prob_bound(z64, y, logp, top, log_sum)
    got, norm = dp.log_prob(z, yd)
    near(got, logp, dl, "log_prob")
    near(norm[:, 0], top, 0.0, "norm maximum")
    near(norm[:, 1], log_sum, dl, "norm log-sum")

    c = rng.standard_normal(rows).astype(np.float32)
    c[rng.random(rows) < 0.1] = 0.0
    g, h = ref64.grad_rows(z64, y, p, c.astype(np.float64), live, none)
    dg, dh = ref64.grad_bound(z64, top, p, c, 0.0, g, h, dtype)
    target = z.clone() if not in_place else None
    if in_place:  # the margins' own storage, strides and all
        keep = z.clone()
        target = z
    gg, hh = dp.log_prob_grad(z, yd, norm, torch.from_numpy(c).cuda(), grad=target, hess=hess)
    near(gg, g, dg, "log_prob_grad")
    if hess:
        near(hh, h, dh, "log_prob_grad curvature")
    if in_place:
        z.copy_(keep)

    old = (np.where(np.isfinite(logp), logp, -3.0) + 0.2 * rng.standard_normal(rows)).astype(np.float32)
    refl = (np.where(np.isfinite(logp), logp, -3.0) + 0.5 * rng.standard_normal(rows)).astype(np.float32)
    adv = rng.standard_normal(rows).astype(np.float32)
    f64 = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    up = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    # the clip bounds, kl are fp32 where the kernel sees them
    clip = tuple(float(np.float32(v)) for v in CLIP)
    kl = float(np.float32(KL))
    for use_ref in (True, False):
        loss, c, size, edge, ratio = ref64.policy(logp, f64(old), f64(adv), f64(refl) if use_ref else None, f64(weight),
                                                  clip, kl)
        skip = ~live | none
        loss, c, size = (np.where(skip, 0.0, v) for v in (loss, c, size))
        # exp(log p - old) is off by log p's error and a few roundings, of the subtraction among them
        rel = dl + ref64.EPS * (8 + np.abs(np.where(np.isfinite(logp), logp, 0.0)) + np.abs(old) + np.abs(refl))
        err = size * 2 * rel + 1e-38
        sure = skip | (edge > 4 * rel * np.maximum(ratio, 1.0))
        assert rows < 10 or sure.mean() > 0.9
        g, h = ref64.grad_rows(z64, y, p, c, live, none)
        dg, dh = ref64.grad_bound(z64, top, p, c, err, g, h, dtype)
        r = dp.policy_loss(z, yd, up(old), up(adv), ref_log_prob=up(refl) if use_ref else None, weight=up(weight),
                           clip=CLIP, kl=KL, hess=hess)
        near(r.log_prob, logp, dl, "policy log_prob")
        near(r.loss, loss, err, "policy loss")
        at = torch.from_numpy(sure).cuda()
        near(r.grad[at], g[sure], dg[sure], "policy gradient")
        if hess:
            near(r.hess[at], h[sure], dh[sure], "policy curvature")
        else:
            assert r.hess is None
        forward = dp.policy_loss(z, yd, up(old), up(adv), ref_log_prob=up(refl) if use_ref else None,
                                 weight=up(weight), clip=CLIP, kl=KL, grad=False)
        assert forward.grad is None and torch.equal(forward.loss, r.loss)
        again = dp.policy_loss(z, yd, up(old), up(adv), ref_log_prob=up(refl) if use_ref else None, weight=up(weight),
                               clip=CLIP, kl=KL, hess=hess)
        assert torch.equal(again.grad, r.grad) and torch.equal(again.loss, r.loss)
        if in_place:
            keep = z.clone()
            into = dp.policy_loss(z, yd, up(old), up(adv), ref_log_prob=up(refl) if use_ref else None,
                                  weight=up(weight), clip=CLIP, kl=KL, grad=z)
            assert into.grad is z and torch.equal(z, r.grad)
            z.copy_(keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 20, 21, 24, 25, 28, 29, 31,
                                     32, 33, 36, 37, 40, 41, 47, 48, 49, 56, 57, 63, 64, 65, 96, 100, 127, 128, 129, 255,
                                     256, 257, 511, 513, 1000, 1024, 1025])
def test_small_class_counts(dp, dtype, classes):
    rows = 203 if classes < 200 else 37
    for pad, shift in ((0, 0), (0, 3), (3, 1), (8, 8)):
        z, z64, rng = margins(rows, classes, dtype, classes * 16 + pad, pad, shift)
        check_rows(dp, z, z64, labels(rng, rows, classes), rng, dtype, hess=pad != 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [2047, 2048, 2049, 4096, 4099, 8191, 8192, 8200, 16384, 16389, 32768, 32775, 65536,
                                     65537, 131072, 131081, 262144, 262151, 300007])
def test_large_class_counts(dp, dtype, classes):
    rows = 5
    for pad, shift in ((0, 0), (1, 5)):
        z, z64, rng = margins(rows, classes, dtype, classes + pad, pad, shift)
        check_rows(dp, z, z64, labels(rng, rows, classes), rng, dtype, hess=pad == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [0, 1, 2, 3, 31, 33, 149, 300, 1000])
@pytest.mark.parametrize("classes", [3, 40, 700, 5003])
def test_row_counts(dp, dtype, rows, classes):
    z, z64, rng = margins(rows, classes, dtype, rows + classes)
    weight = rng.random(rows).astype(np.float32)
    weight[rng.random(rows) < 0.2] = 0.0
    check_rows(dp, z, z64, labels(rng, rows, classes), rng, dtype, weight=weight)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [24, 40, 64, 65, 72, 96, 127, 128, 160, 200, 256, 257, 320, 500, 512, 640, 1000, 1024])
def test_many_rows(dp, dtype, classes):
    """Rows past the count where each gets a warp: 2 to 32 lanes a row."""
    rows = 2501
    for pad, shift in ((0, 0), (5, 2)) if classes < 300 else ((0, 0),):
        z, z64, rng = margins(rows, classes, dtype, 3 * classes + pad, pad, shift)
        check_rows(dp, z, z64, labels(rng, rows, classes), rng, dtype, hess=classes % 3 != 0, in_place=pad > 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,pad", [(3600, 2051, 0), (1800, 4104, 3), (900, 8208, 0), (460, 16400, 1)])
def test_many_long_rows(dp, dtype, rows, classes, pad):
    """As many rows as fill the device with 32, 64 and 128 threads a row, runs
    of skipped rows among them."""
    z, z64, rng = margins(rows, classes, dtype, rows + pad, pad, pad)
    y = labels(rng, rows, classes)
    y[rows // 3: rows // 2] = -1
    check_rows(dp, z, z64, y, rng, dtype, hess=False, in_place=pad > 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 33, 129, 1001, 9000, 70001])
def test_gradient_in_the_margins_place(dp, dtype, classes):
    for pad, shift in ((0, 0), (5, 2)):
        z, z64, rng = margins(21, classes, dtype, classes, pad, shift)
        check_rows(dp, z, z64, labels(rng, 21, classes), rng, dtype, hess=False, in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [6, 90, 1500, 20011, 140001])
def test_masked_classes_and_rows(dp, dtype, classes):
    """-inf and the type's lowest value as masks: a few classes left, one left,
    none left; and margins far from zero."""
    rows = 24
    z, z64, rng = margins(rows, classes, dtype, 5 * classes, 2, 1)
    lowest = float(torch.finfo(z.dtype).min)
    y = rng.integers(0, classes, rows).astype(np.int32)
    for r in range(rows):
        kind = r % 8
        masked = np.ones(classes, bool) if kind in (1, 2, 6, 7) else rng.random(classes) < 0.7
        if kind in (0, 1, 3):
            masked[y[r]] = False           # the label's class stays
        value = -np.inf if kind in (0, 1, 2) else lowest
        if kind != 5:
            z64[r, masked] = value         # kind 2: no class; kinds 6, 7: every margin the lowest value
        else:
            z64[r] += 400.0 if dtype != "float32" else 3000.0
    z.copy_(torch.from_numpy(z64).to(z.dtype))
    z64 = z.double().cpu().numpy()
    # a masked label's log p is -inf or about the type's lowest value, and the
    # loss's KL term infinite by its formula: those rows go without a label,
    # unless every class is masked alike
    chosen = z64[np.arange(rows), y]
    hidden = ((chosen == -np.inf) | (chosen == lowest)) & (z64.max(1) > chosen)
    y[hidden] = -1
    check_rows(dp, z, z64, y, rng, dtype)


@pytest.mark.parametrize("classes", [4, 60, 600, 6000, 60000])
def test_nan_and_infinity_stay_in_their_rows(dp, classes):
    rows = 12
    z, z64, rng = margins(rows, classes, "float32", classes)
    y = rng.integers(0, classes, rows).astype(np.int32)
    clean = torch.from_numpy(z64).float().cuda()
    yd = torch.from_numpy(y).cuda()
    old = torch.zeros(rows, device="cuda") - 3
    adv = torch.ones(rows, device="cuda")
    base = dp.policy_loss(clean, yd, old, adv, hess=True)
    z[1, classes // 2] = float("nan")
    z[4, classes - 1] = float("inf")
    z[6] = float("nan")
    z[8] = float("nan")
    yd[8] = -1  # a skipped row's margins are not looked at
    weight = torch.ones(rows, device="cuda")
    z[10] = float("nan")
    weight[10] = 0  # nor do they count in a row of weight 0
    r = dp.policy_loss(z, yd, old, adv, weight=weight, hess=True)
    bad = [1, 4, 6]
    fine = [i for i in range(rows) if i not in bad + [8, 10]]
    for a, b in ((r.loss, base.loss), (r.log_prob, base.log_prob), (r.grad, base.grad), (r.hess, base.hess)):
        assert torch.equal(a[fine], b[fine])
    assert torch.isnan(r.loss[bad]).all() and torch.isnan(r.log_prob[bad]).all() and torch.isnan(r.grad[bad]).all()
    assert (r.loss[[8, 10]] == 0).all() and (r.grad[[8, 10]] == 0).all() and (r.hess[[8, 10]] == 0).all()
    logp, norm = dp.log_prob(z, yd)
    c = torch.ones(rows, device="cuda")
    c[10] = 0
    g, h = dp.log_prob_grad(z, yd, norm, c, hess=True)
    assert torch.isnan(logp[bad]).all() and torch.isnan(g[bad]).all()
    assert torch.isfinite(g[fine]).all() and (g[[8, 10]] == 0).all() and (h[[8, 10]] == 0).all()
    assert logp[8] == 0 and (norm[8] == 0).all()


def test_offsets_past_32_bits(dp):
    """Rows more than 2^31 elements apart: offsets are 64-bit in every kernel."""
    for classes in (8, 100, 3001):
        apart = (1 << 31) + 24
        store = torch.empty(2 * apart + classes, dtype=torch.bfloat16, device="cuda")
        z = store.as_strided((3, classes), (apart, 1))
        small, z64, rng = margins(3, classes, "bfloat16", classes)
        z.copy_(small)
        y = torch.from_numpy(rng.integers(0, classes, 3).astype(np.int32)).cuda()
        c = torch.tensor([1.0, -0.5, 2.0], device="cuda")
        a, na = dp.log_prob(small, y)
        b, nb = dp.log_prob(z, y)
        near(b, a.double().cpu().numpy(), 1e-5, "log_prob")
        ga, _ = dp.log_prob_grad(small, y, na, c)
        gb, _ = dp.log_prob_grad(z, y, nb, c, grad=z)
        near(gb, ga.double().cpu().numpy(), 2.0 ** -7, "gradient")
        del store, z
        torch.cuda.empty_cache()


def test_another_stream(dp):
    z, z64, rng = margins(500, 3000, "float32", 9)
    y = torch.from_numpy(labels(rng, 500, 3000)).cuda()
    want, norm = dp.log_prob(z, y)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        z2 = z + 0.0  # made late on this stream: a call on another one would read what was there before
        got, n2 = dp.log_prob(z2, y)
        g2, _ = dp.log_prob_grad(z2, y, n2, want)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(n2, norm)
    g, _ = dp.log_prob_grad(z, y, norm, want)
    assert torch.equal(g, g2)


def test_calls_can_be_captured_in_a_graph(dp):
    z, z64, rng = margins(64, 5000, "bfloat16", 4)
    y = torch.from_numpy(labels(rng, 64, 5000)).cuda()
    begin = torch.arange(0, 65, 8, device="cuda")[:9]

    def step():
        logp, norm = dp.log_prob(z, y)
        r = dp.preference_loss(logp, item_begin=begin, beta=0.1)
        return r.loss, dp.log_prob_grad(z, y, norm, r.grad)[0]
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_log_prob_gradient_is_the_softmax_objectives(dp):
    """c = -1: the cross-entropy gradient that dp_gradients computes."""
    rows, classes = 3000, 5
    z, z64, rng = margins(rows, classes, "float32", 2)
    y = rng.integers(0, classes, rows).astype(np.int32)
    yd = torch.from_numpy(y).cuda()
    _, norm = dp.log_prob(z, yd)
    g, h = dp.log_prob_grad(z, yd, norm, torch.full((rows,), -1.0, device="cuda"), hess=True)
    gh = torch.empty((classes, rows, 2), device="cuda")
    scales = torch.empty((classes, 2), device="cuda")
    zc, yf = z.contiguous(), yd.float()
    dp.check(dp.lib().dp_gradients(2, classes, zc.data_ptr(), yf.data_ptr(), rows, gh.data_ptr(), scales.data_ptr(), None))
    assert torch.allclose(g, gh[:, :, 0].T, rtol=0, atol=2e-6)
    assert torch.allclose(h, gh[:, :, 1].T, rtol=0, atol=2e-6)


def test_policy_gradient_against_differences(dp):
    """Central differences of the kernel's own loss: step 2^-5, so the third
    derivative's term is below 2^-10 of the weight's scale and the loss's
    rounding below 2^-18 / 2^-5."""
    rows, classes, step = 6, 7, 2.0 ** -5
    z, z64, rng = margins(rows, classes, "float32", 3, scale=1.0)
    y = torch.from_numpy(rng.integers(0, classes, rows).astype(np.int32)).cuda()
    logp, _ = dp.log_prob(z, y)
    old = logp + torch.tensor([0.05, -0.05, 0.0, 0.1, -0.1, 0.02], device="cuda")  # ratios inside the clip range
    refl = logp + 0.3
    adv = torch.tensor([1.0, -1.0, 0.5, 2.0, -2.0, 0.7], device="cuda")
    f = lambda t: dp.policy_loss(t, y, old, adv, ref_log_prob=refl, clip=(0.5, 0.5), kl=0.2)  # noqa: E731
    g = f(z).grad
    for k in range(classes):
        up, down = z.clone(), z.clone()
        up[:, k] += step
        down[:, k] -= step
        slope = (f(up).loss.double() - f(down).loss.double()) / (2 * step)
        assert (slope - g[:, k].double()).abs().max() < 2e-3


# ---------------------------------------------------------------- preference

def pair_bound(x, terms, w, beta, x_err):
    """The terms' derivatives are at most 1, 1/4 and 1/10 in size, each is
    rounded a few times, and the loss is as large as x."""
    loss, slope, bend = terms
    e = ref64.EPS * 16
    return (w * (x_err + e * (np.abs(loss) + 1e-30)), w * beta * (x_err / 4 + e * np.abs(slope)) + 1e-37,
            w * beta * beta * (x_err / 8 + e * bend) + 1e-37)


@pytest.mark.parametrize("use_ref", [False, True])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("lengths", ["one", "short", "few", "uneven", "mixed", "long", "empty", "huge", "ragged", "wide"])
def test_preference_over_segments(dp, lengths, smoothing, use_ref):
    rng = np.random.default_rng(7)
    items = {"one": 4000, "short": 600, "few": 9000, "uneven": 5000, "mixed": 200, "long": 6, "empty": 50, "huge": 2, "ragged": 10,
             "wide": 6}[lengths]
    n = {"one": np.ones(items, int), "short": rng.integers(1, 9, items), "few": rng.integers(0, 9, items),
         "uneven": np.where(rng.random(items) < 0.002, 3000, rng.integers(0, 4, items)), "mixed": rng.integers(0, 700, items),
         "long": rng.integers(3000, 9000, items), "empty": rng.integers(0, 2, items),
         "huge": np.array([300_001, 77_777]),
         "wide": rng.integers(20_000, 60_000, items),
         "ragged": np.array([0, 1_000_003, 3, 0, 150_000, 8191, 60_000, 250_001, 16_385, 0])}[lengths]
    lead, tail = (0, 0) if lengths == "one" else (3, 5)
    begin = lead + np.concatenate([[0], np.cumsum(n)])
    rows = int(begin[-1]) + tail
    spread = 2.0 / np.sqrt(max(1.0, n.mean()))
    score = (rng.standard_normal(rows) * spread).astype(np.float32)
    refs = (rng.standard_normal(rows) * spread).astype(np.float32) if use_ref else None
    w = rng.random(items // 2).astype(np.float32)
    w[::5] = 0.0
    beta, smooth = float(np.float32(0.7)), float(np.float32(smoothing))
    gap = score.astype(np.float64) - (refs.astype(np.float64) if use_ref else 0.0)
    total = ref64.item_sums(gap, begin)
    x = beta * (total[0::2] - total[1::2])
    terms = ref64.pair_terms(x, smooth)
    size = ref64.item_sums(np.abs(gap), begin)
    x_err = beta * ref64.EPS * (4 + 12 + n.max() / 32) * (size[0::2] + size[1::2]) + 4 * ref64.EPS * np.abs(x)
    bl, bs, bb = pair_bound(x, terms, w, beta, x_err)
    up = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    give = None if lengths == "one" else up(begin)
    r = dp.preference_loss(up(score), ref_score=up(refs), item_begin=give, weight=up(w), beta=beta, smoothing=smooth,
                           hess=True)
    near(r.loss, w * terms[0], bl, "loss")
    q, k = w * beta * terms[1], np.maximum(w * beta * beta * terms[2], 1e-16)
    rowwise = lambda a, b, out: np.concatenate([np.full(lead, out), np.repeat(np.stack([a, b], 1).reshape(-1), n),  # noqa: E731
                                                np.full(tail, out)])
    near(r.grad, rowwise(q, -q, 0.0), rowwise(bs, bs, 0.0), "gradient")
    near(r.hess, rowwise(k, k, 1e-16), rowwise(bb, bb, 0.0) + 1e-22, "curvature")
    plain = dp.preference_loss(up(score), ref_score=up(refs), item_begin=give, weight=up(w), beta=beta, smoothing=smooth)
    assert plain.hess is None and torch.equal(plain.grad, r.grad)


def pair_case(kind, rng):
    if kind == "few":
        rows, pairs = 5, np.array([[0, 1], [1, 2], [3, 1], [0, 1]])
    elif kind == "none":
        rows, pairs = 7, np.zeros((0, 2), int)
    elif kind == "star":          # one row against all the others
        rows = 20_001
        pairs = np.stack([np.zeros(rows - 1, int), np.arange(1, rows)], 1)
        pairs[::3] = pairs[::3, ::-1]
    elif kind == "groups":        # every two rows of a group
        rows, size = 960, 12
        i, j = np.triu_indices(size, 1)
        pairs = np.concatenate([np.stack([i, j], 1) + g * size for g in range(rows // size)])
    elif kind == "skewed":
        rows = 3000
        a = np.minimum((rows * rng.random(60_000) ** 6).astype(int), rows - 1)
        pairs = np.stack([a, (a + rng.integers(1, rows, len(a))) % rows], 1)
    else:
        rows = 50_000
        a = rng.integers(0, rows, 40_000)
        pairs = np.stack([a, (a + rng.integers(1, rows, len(a))) % rows], 1)
    return rows, pairs.astype(np.int32)


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("kind", ["few", "none", "star", "groups", "skewed", "sparse"])
def test_preference_over_any_pairs(dp, kind, weighted):
    rng = np.random.default_rng(11)
    rows, pairs = pair_case(kind, rng)
    score = (2 * rng.standard_normal(rows)).astype(np.float32)
    refs = rng.standard_normal(rows).astype(np.float32) if weighted else None
    w = rng.random(len(pairs)).astype(np.float32) if weighted else None
    beta, smooth = float(np.float32(1.3)), float(np.float32(0.05))
    gap = score.astype(np.float64) - (refs if weighted else 0.0)
    a, b = pairs[:, 0], pairs[:, 1]
    x = beta * (gap[a] - gap[b])
    terms = ref64.pair_terms(x, smooth)
    w64 = w.astype(np.float64) if weighted else np.ones(len(pairs))
    x_err = beta * ref64.EPS * 8 * (np.abs(gap[a]) + np.abs(gap[b])) + 4 * ref64.EPS * np.abs(x)
    bl, bs, bb = pair_bound(x, terms, w64, beta, x_err)
    q, k = w64 * beta * terms[1], w64 * beta * beta * terms[2]
    count = np.bincount(a, minlength=rows) + np.bincount(b, minlength=rows)
    total = lambda u, v: np.bincount(a, u, rows) + np.bincount(b, v, rows)  # noqa: E731
    chain = ref64.EPS * (64 + np.minimum(count, 4096))  # a row's sum: chains of at most 4096 terms, then a tree
    up = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    plan = dp.PreferencePairs(up(pairs), rows)
    r = plan.loss(up(score), ref_score=up(refs), weight=up(w), beta=beta, smoothing=smooth, hess=True)
    near(r.loss, w64 * terms[0], bl, "loss")
    near(r.grad, total(q, -q), total(bs, bs) + chain * total(np.abs(q), np.abs(q)) + 1e-37, "gradient")
    near(r.hess, np.maximum(total(k, k), 1e-16), total(bb, bb) + chain * total(k, k) + 1e-22, "curvature")
    again = plan.loss(up(score), ref_score=up(refs), weight=up(w), beta=beta, smoothing=smooth, hess=True)
    assert all(torch.equal(u, v) for u, v in zip(r, again))
    other = dp.PreferencePairs(up(pairs), rows).loss(up(score), ref_score=up(refs), weight=up(w), beta=beta,
                                                     smoothing=smooth)
    assert torch.equal(other.grad, r.grad) and other.hess is None
    plan.free()
    with pytest.raises(dp.DPError, match="freed"):
        plan.loss(up(score))


def test_pairs_agree_with_segments(dp):
    rows = 2000
    score = torch.randn(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    pairs = torch.arange(rows, dtype=torch.int32, device="cuda").view(-1, 2)
    a = dp.preference_loss(score, beta=0.5, smoothing=0.2, hess=True)
    b = dp.PreferencePairs(pairs, rows).loss(score, beta=0.5, smoothing=0.2, hess=True)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_weightless_pairs_and_infinite_scores(dp):
    score = torch.tensor([float("nan"), 1.0, float("inf"), 0.0, 0.0, float("inf"), 1e30, -1e30], device="cuda")
    weight = torch.tensor([0.0, 1.0, 1.0, 1.0], device="cuda")
    pairs = torch.arange(8, dtype=torch.int32, device="cuda").view(-1, 2)
    for r in (dp.preference_loss(score, weight=weight, hess=True),
              dp.PreferencePairs(pairs, 8).loss(score, weight=weight, hess=True)):
        assert r.loss.tolist() == [0.0, 0.0, float("inf"), 0.0]
        assert r.grad.tolist() == [0.0, 0.0, 0.0, 0.0, -1.0, 1.0, 0.0, 0.0]
        assert (r.hess == torch.tensor(1e-16, device="cuda")).all()


def test_preference_gradient_against_differences(dp):
    step = 2.0 ** -5
    score = torch.tensor([0.3, -0.2, 1.1, 0.4, 0.0, -0.7], device="cuda")
    pairs = torch.tensor([[0, 1], [2, 1], [3, 4], [5, 0], [2, 5]], dtype=torch.int32, device="cuda")
    plan = dp.PreferencePairs(pairs, 6)
    f = lambda s: plan.loss(s, beta=0.8, smoothing=0.1, hess=True)  # noqa: E731
    r = f(score)
    for i in range(6):
        up, down = score.clone(), score.clone()
        up[i] += step
        down[i] -= step
        a, b = f(up).loss.double().sum(), f(down).loss.double().sum()
        assert abs((a - b) / (2 * step) - r.grad[i].double()) < 1e-3
        slope = (f(up).grad[i].double() - f(down).grad[i].double()) / (2 * step)
        assert abs(slope - r.hess[i].double()) < 1e-3


def test_bad_pairs_are_refused(dp):
    for rows, pairs, what in ((4, [[0, 4]], "outside"), (4, [[-1, 2]], "outside"), (4, [[0, 1], [2, 2]], "twice")):
        with pytest.raises(dp.DPError, match=what):
            dp.PreferencePairs(torch.tensor(pairs, dtype=torch.int32, device="cuda"), rows)


def test_binding_refusals(dp):
    z = torch.zeros(4, 6, device="cuda")
    y = torch.zeros(4, dtype=torch.int32, device="cuda")
    one = torch.zeros(4, device="cuda")
    _, norm = dp.log_prob(z, y)
    store = torch.zeros(64, device="cuda")
    cases = [
        (lambda: dp.log_prob(z.double(), y), "float32, float16 or bfloat16"),
        (lambda: dp.log_prob(z.t(), y[:1].expand(6)), "adjacent"),
        (lambda: dp.log_prob(z[0], y), "rows, classes"),
        (lambda: dp.log_prob(z, y.long()), "int32"),
        (lambda: dp.log_prob(z, y[:3]), "shape"),
        (lambda: dp.log_prob(z, y.cpu()), "must be on"),
        (lambda: dp.log_prob(z.cpu(), y), "CUDA"),
        (lambda: dp.log_prob(z[:1].expand(4, 6), y), "stride must cover"),
        (lambda: dp.log_prob_grad(z, y, norm[:, 0], one), "shape"),
        (lambda: dp.log_prob_grad(z, y, norm, one, grad=z.half()), "margins' shape, type"),
        (lambda: dp.log_prob_grad(store[:24].view(4, 6), y, norm, one, grad=store[2:26].view(4, 6)), "overlap"),
        (lambda: dp.policy_loss(z, y, one, one, clip=(1.5, 0.2)), "clip_low"),
        (lambda: dp.policy_loss(z, y, one, one, clip=(0.2, float("inf"))), "clip_high"),
        (lambda: dp.policy_loss(z, y, one, one, kl=-1.0), "KL"),
        (lambda: dp.policy_loss(z, y, one, one, grad=False, hess=True), "hess"),
        (lambda: dp.preference_loss(one[:3]), "pairs of rows"),
        (lambda: dp.preference_loss(one, beta=0.0), "beta"),
        (lambda: dp.preference_loss(one, smoothing=0.7), "smoothing"),
        (lambda: dp.preference_loss(one, item_begin=torch.zeros(4, dtype=torch.int64, device="cuda")), "offsets"),
    ]
    for call, what in cases:
        with pytest.raises(dp.DPError, match=what):
            call()
