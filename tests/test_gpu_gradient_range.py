"""Boosting rounds on gradients of any finite size, and of sizes far apart."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("power", [64, 99, 101, 114, 125])
@pytest.mark.parametrize("scaled_hess", [False, True])
def test_trees_scale_with_the_gradients(dp, power, scaled_hess):
    """Powers of two in all gradients (and curvatures) change no split, and the
    leaves by the same power alone: each step of a round is exact in them."""
    rows = 40_000  # more than two windows of 16,383
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((rows, 5), dtype=np.float32)).cuda()
    d = dp.DMatrix.from_torch(x)
    g = (x[:, 0] + 0.3 * x[:, 1].sign() + 1.0).clamp(-3.9, 3.9)
    h = torch.rand(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(0)) + 0.5
    # (curvatures scaled too: no regularisation, so that their power cancels)
    params = {"objective": "reg:squarederror", "max_depth": 4, "base_score": 0, "eta": 0.5,
              "lambda": 0 if scaled_hess else 1, "min_child_weight": 0}
    trees = []
    for k in (0, power):
        b = dp.Booster(params, [d])
        b.boost(d, 0, g * 2.0 ** k, h * 2.0 ** (k if scaled_hess else 0))
        trees.append(b.trees()[0])
    small, large = trees
    for f in ("left_children", "right_children", "split_indices", "default_left"):
        assert small[f] == large[f], f
    assert len(small["left_children"]) > 15
    by = 0 if scaled_hess else power
    inner = np.array(small["left_children"]) >= 0
    for f, scaled in (("base_weights", np.full(len(inner), True)), ("split_conditions", ~inner)):  # (a leaf's condition is its value)
        u, v = (np.array(t[f], np.float32) for t in trees)  # (the model's text is fp32's shortest)
        assert np.array_equal(v, np.where(scaled, np.ldexp(u, by), u)), f


@pytest.mark.parametrize("power,kept", [(10, True), (20, False)])
def test_gradients_far_below_the_largest(dp, power, kept):
    """Steps are at least 2^-17 and at most 2^-16 of the largest: next to one of
    2^10 gradients of 1 keep three digits, next to one of 2^20 they count as 0."""
    rows = 2000
    x = torch.zeros(rows, 1, device="cuda")
    x[rows // 2:] = 1.0
    g = torch.ones(rows, device="cuda") * 1.1
    g[0] = 2.0 ** power
    d = dp.DMatrix.from_torch(x)
    b = dp.Booster({"objective": "reg:squarederror", "max_depth": 1, "base_score": 0, "eta": 1.0, "lambda": 0}, [d])
    b.boost(d, 0, g, torch.ones(rows, device="cuda"))
    t = b.trees()[0]
    assert t["left_children"][0] == 1
    right = t["base_weights"][t["right_children"][0]]
    assert abs(right + 1.1) <= 2.0 ** (power - 17) if kept else right == 0
