"""Argument checks of the choice losses' C entry points, which come before any
device work, and their 64-bit formulas against differences (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import loss_reference as ref64

A = 4096  # an aligned address that no refused call reads


def refused(dp, name, *args):
    assert getattr(dp.lib(), name)(*args) == -1
    return dp.lib().XGBGetLastError().decode()


@pytest.mark.parametrize("change,what", [
    ({"dtype": 3}, "margin type"), ({"dtype": -1}, "margin type"), ({"classes": 0}, "number of classes"),
    ({"classes": 1 << 31}, "number of classes"), ({"stride": 9}, "cover the classes"),
    ({"stride": (1 << 40) + 1}, "out of range"), ({"rows": 1 << 61}, "overflows"), ({"margin": None}, "margin pointer"),
    ({"margin": A + 2}, "not aligned"), ({"label": None}, "null"),
])
def test_margin_checks(dp, change, what):
    a = {"dtype": 0, "margin": A, "rows": 4, "classes": 10, "stride": 10, "label": A, **change}
    lead = (a["dtype"], a["margin"], a["rows"], a["classes"], a["stride"], a["label"])
    far = 1 << 30
    assert what in refused(dp, "dp_log_prob", *lead, A, A, None)
    assert what in refused(dp, "dp_log_prob_grad", *lead, A, A, far, 10, None, 0, None)
    assert what in refused(dp, "dp_policy_loss", *lead, A, None, A, None, 0.2, 0.2, 0.0, A, A, far, 10, None, 0, None)


def test_output_checks(dp):
    lead = (0, A, 4, 10, 10, A)
    policy = lambda *tail, clip=(0.2, 0.2), kl=0.0, loss=A: refused(  # noqa: E731
        dp, "dp_policy_loss", *lead, A, None, A, None, *clip, kl, loss, A, *tail, None)
    assert "norm pointer is not aligned" in refused(dp, "dp_log_prob", *lead, A, A + 4, None)
    assert "null" in refused(dp, "dp_log_prob", *lead, None, A, None)
    assert "null" in refused(dp, "dp_log_prob_grad", *lead, A, A, None, 10, None, 0, None)
    assert "null" in policy(None, 0, None, 0, loss=None)
    assert "gradient pointer is null" in policy(None, 0, A, 10)
    assert "gradient row stride" in policy(1 << 20, 9, None, 0)
    assert "overlap" in policy(A + 8, 10, None, 0)
    assert "overlap" in policy(A, 12, None, 0)
    assert "curvature overlaps" in policy(1 << 20, 10, A, 10)
    assert "curvature overlaps" in policy(1 << 20, 10, 1 << 20, 10)
    assert "curvature row stride" in policy(1 << 20, 10, 1 << 22, 4)
    for clip, kl, what in (((-0.1, 0.2), 0.0, "clip_low"), ((1.1, 0.2), 0.0, "clip_low"),
                           ((float("nan"), 0.2), 0.0, "clip_low"), ((0.2, -1.0), 0.0, "clip_high"),
                           ((0.2, float("nan")), 0.0, "clip_high"), ((0.2, 0.2), -1.0, "KL"),
                           ((0.2, 0.2), float("inf"), "KL")):
        assert what in policy(1 << 20, 10, None, 0, clip=clip, kl=kl)


def test_preference_checks(dp):
    call = lambda rows, begin, pairs, beta=1.0, smooth=0.0, score=A, loss=A, grad=A: refused(  # noqa: E731
        dp, "dp_preference_loss", rows, begin, pairs, score, None, None, beta, smooth, loss, grad, None, None)
    assert "two rows" in call(7, None, 4)
    assert "null" in call(8, None, 4, score=None)
    assert "null" in call(8, None, 4, grad=None)
    assert "loss pointer" in call(8, None, 4, loss=None)
    for beta in (0.0, -1.0, float("nan"), float("inf")):
        assert "beta" in call(8, None, 4, beta=beta)
    for smooth in (-0.1, 0.6, float("nan")):
        assert "smoothing" in call(8, None, 4, smooth=smooth)
    plan = C.c_void_p()
    assert "below 2^31" in refused(dp, "dp_preference_prepare", 1 << 31, A, 4, None, C.byref(plan))
    assert "below 2^31" in refused(dp, "dp_preference_prepare", 4, A, 1 << 31, None, C.byref(plan))
    assert "null" in refused(dp, "dp_preference_prepare", 4, None, 4, None, C.byref(plan))
    assert "output pointer" in refused(dp, "dp_preference_prepare", 4, A, 4, None, None)
    assert "plan is null" in refused(dp, "dp_preference_run", None, A, None, None, 1.0, 0.0, A, A, None, None)
    assert not plan.value
    assert dp.lib().dp_preference_free(None) == 0


def test_vectors_off_their_boundaries(dp):
    odd = A + 2
    lead = (0, A, 4, 10, 10)
    for label, out in ((odd, A), (A, odd)):
        assert "not aligned" in refused(dp, "dp_log_prob", *lead, label, out, A, None)
    assert "not aligned" in refused(dp, "dp_log_prob_grad", *lead, A, A, odd, 1 << 20, 10, None, 0, None)
    assert "not aligned" in refused(dp, "dp_policy_loss", *lead, A, A, None, odd, None, 0.2, 0.2, 0.0, A, A, None, 0,
                                    None, 0, None)
    assert "not aligned" in refused(dp, "dp_preference_loss", 8, None, 4, odd, None, None, 1.0, 0.0, A, A, None, None)
    assert "not aligned" in refused(dp, "dp_preference_loss", 8, A + 4, 4, A, None, None, 1.0, 0.0, A, A, None, None)
    plan = C.c_void_p()
    assert "not aligned" in refused(dp, "dp_preference_prepare", 4, odd, 4, None, C.byref(plan))


def test_no_rows_need_no_device(dp):
    assert dp.lib().dp_log_prob(0, None, 0, 10, 10, None, None, None, None) == 0
    assert dp.lib().dp_log_prob_grad(2, None, 0, 10, 10, None, None, None, None, 10, None, 0, None) == 0
    assert dp.lib().dp_policy_loss(1, None, 0, 10, 10, None, None, None, None, None, 0.2, 0.2, 0.0, None, None, None, 0,
                                   None, 0, None) == 0
    assert dp.lib().dp_preference_loss(0, None, 0, None, None, None, 1.0, 0.0, None, None, None, None) == 0


def test_training_on_caller_gradients_checks(dp):
    b = dp.Booster({"objective": "multi:softprob", "num_class": 3})
    text = dp.array_interface(A, [4, 3]).encode()
    assert "Booster handle" in refused(dp, "XGBoosterTrainOneIter", None, None, 0, text, text)
    assert "DMatrix handle" in refused(dp, "XGBoosterTrainOneIter", b.handle, None, 0, text, text)
    n, p = C.c_uint64(), C.c_void_p()
    assert "output pointer" in refused(dp, "dp_booster_train_margin", b.handle, None, None, C.byref(n), C.byref(p))
    assert "DMatrix handle" in refused(dp, "dp_booster_train_margin", b.handle, None, C.byref(n), C.byref(n), C.byref(p))


def test_formulas_against_differences():
    rng = np.random.default_rng(0)
    z = rng.standard_normal((5, 6))
    y = rng.integers(0, 6, 5)
    old, refs, adv = (rng.standard_normal(5) * s - o for s, o in ((0.05, 1.8), (0.3, 1.8), (1.0, 0.0)))
    w = rng.random(5)
    logp = lambda v: ref64.softmax_rows(v, y)[0]  # noqa: E731
    old = logp(z) + 0.05 * rng.standard_normal(5)
    loss = lambda v: ref64.policy(logp(v), old, adv, refs, w, (0.4, 0.4), 0.1)[0]  # noqa: E731
    _, top, log_sum, p, live, none = ref64.softmax_rows(z, y)
    g, _ = ref64.grad_rows(z, y, p, ref64.policy(logp(z), old, adv, refs, w, (0.4, 0.4), 0.1)[1], live, none)
    step = 1e-5
    for k in range(6):
        d = np.zeros_like(z)
        d[:, k] = step
        assert np.allclose((loss(z + d) - loss(z - d)) / (2 * step), g[:, k], atol=1e-8)
    x = np.linspace(-30, 30, 61)
    for smooth in (0.0, 0.1):
        t = ref64.pair_terms(x, smooth)
        up, down = ref64.pair_terms(x + step, smooth), ref64.pair_terms(x - step, smooth)
        assert np.allclose((up[0] - down[0]) / (2 * step), t[1], atol=1e-8)
        assert np.allclose((up[1] - down[1]) / (2 * step), t[2], atol=1e-8)


def test_preference_outputs_may_not_overlap(dp):
    call = lambda grad, hess=None, ref=None: refused(  # noqa: E731
        dp, "dp_preference_loss", 8, None, 4, A, ref, None, 1.0, 0.0, A + 1024, grad, hess, None)
    assert "gradient overlaps" in call(A)
    assert "gradient overlaps" in call(A + 28)
    assert "gradient overlaps" in call(A + 128, ref=A + 156)
    assert "curvature overlaps" in call(A + 128, A)
    assert "curvature overlaps" in call(A + 128, A + 128)
    assert "curvature overlaps" in call(A + 128, A + 256, ref=A + 284)
