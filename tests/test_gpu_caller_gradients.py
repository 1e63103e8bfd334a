"""Boosting rounds on a caller's gradients (XGBoosterTrainOneIter): the same
trees as the objective's own gradients give, and training on the choice
losses end to end."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def table(rows, features, seed=0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(rng.standard_normal((rows, features), dtype=np.float32)).cuda(), rng


def same_trees(a, b):
    ta, tb = a.trees(), b.trees()
    assert len(ta) == len(tb)
    for i, (u, v) in enumerate(zip(ta, tb)):
        for f in ("left_children", "right_children", "split_indices", "split_conditions", "base_weights", "default_left"):
            assert u[f] == v[f], (i, f)


def own_gradients(dp, objective, classes, margin, label):
    rows = margin.shape[0]
    gh = torch.empty((classes, rows, 2), device="cuda")
    scales = torch.empty((classes, 2), device="cuda")
    dp.check(dp.lib().dp_gradients(dp.OBJECTIVE_IDS[objective], classes, margin.data_ptr(), label.data_ptr(), rows,
                                   gh.data_ptr(), scales.data_ptr(), None))
    return gh[:, :, 0].T.contiguous(), gh[:, :, 1].T.contiguous()


@pytest.mark.parametrize("objective,classes", [("reg:squarederror", 1), ("binary:logistic", 1), ("multi:softprob", 3),
                                               ("multi:softprob", 70)])
@pytest.mark.parametrize("subsample", [1.0, 0.6])
def test_same_trees_as_the_objective(dp, objective, classes, subsample):
    x, rng = table(5003, 9)
    y = torch.from_numpy(rng.integers(0, max(classes, 2), 5003).astype(np.float32)).cuda()
    params = {"objective": objective, "max_depth": 4, "eta": 0.4, "subsample": subsample, "seed": 3}
    if classes > 1:
        params["num_class"] = classes
    d, bare = dp.DMatrix.from_torch(x, y), dp.DMatrix.from_torch(x)
    want = dp.train(params, d, 4)
    got = dp.Booster(params, [bare])
    for i in range(4):
        g, h = own_gradients(dp, objective, classes, got.train_margin(bare), y)
        wide = torch.zeros((5003, 2 * classes + 1), device="cuda")  # rows with a stride
        wide[:, :classes] = g
        got.boost(bare, i, wide[:, :classes], h if classes > 1 else h[:, 0])
    same_trees(want, got)
    # rounds of both kinds may alternate
    mixed = dp.Booster(params, [d])
    for i in range(4):
        if i in (0, 3):
            mixed.update(d, i)
        else:
            mixed.boost(d, i, *own_gradients(dp, objective, classes, mixed.train_margin(d), y))
    same_trees(want, mixed)
    assert np.array_equal(mixed.margins(5003, classes), mixed.train_margin(d).cpu().numpy())


def test_refused_gradients_leave_the_model(dp):
    x, _ = table(300, 4)
    d = dp.DMatrix.from_torch(x)
    b = dp.Booster({"objective": "reg:squarederror", "max_depth": 3}, [d])
    one = torch.ones(300, device="cuda")
    b.boost(d, 0, torch.linspace(-1, 1, 300, device="cuda"), one)
    before = b.save_raw()
    for bad in (float("nan"), float("inf")):
        g = torch.zeros(300, device="cuda")
        g[299] = bad
        with pytest.raises(dp.DPError, match="finite"):
            b.boost(d, 1, g, one)
        with pytest.raises(dp.DPError, match="finite"):
            b.boost(d, 1, one, g)
    with pytest.raises(dp.DPError, match="negative"):
        b.boost(d, 1, one, -one)
    for g, h, what in ((one[:299], one, "one row for every row"), (one, torch.ones(300, 2, device="cuda"), "shape"),
                       (one.double(), one, "float32"), (one.cpu(), one, "CUDA"),
                       (one[:1].expand(300), one, "stride must cover")):
        with pytest.raises(dp.DPError, match=what):
            b.boost(d, 1, g, h)
    with pytest.raises(dp.DPError, match="no labels"):
        b.update(d, 1)
    assert b.save_raw() == before and b.boosted_rounds() == 1
    b.boost(d, 1, torch.linspace(-1, 1, 300, device="cuda"), one)
    assert b.boosted_rounds() == 2


def test_ranking_from_preferences(dp):
    """Scores learned from pairs of rows alone order the rows as the hidden score does."""
    rows = 4000
    x, rng = table(rows, 6, 1)
    hidden = (x[:, 0] + 0.5 * x[:, 1] * x[:, 2]).cpu().numpy()
    a = rng.integers(0, rows, 30_000)
    b = (a + rng.integers(1, rows, len(a))) % rows
    wins = hidden[a] > hidden[b]
    pairs = np.where(wins[:, None], np.stack([a, b], 1), np.stack([b, a], 1)).astype(np.int32)
    plan = dp.PreferencePairs(torch.from_numpy(pairs).cuda(), rows)
    d = dp.DMatrix.from_torch(x)
    model = dp.Booster({"objective": "reg:squarederror", "max_depth": 5, "eta": 0.3, "base_score": 0}, [d])
    losses = []
    for i in range(30):
        r = plan.loss(model.train_margin(d)[:, 0], hess=True)
        losses.append(r.loss.mean().item())
        model.boost(d, i, r.grad, r.hess)
    assert abs(losses[0] - np.log(2)) < 1e-6 and losses[-1] < 0.25
    score = model.predict(x, margin=True)[:, 0].cpu().numpy()
    assert (score[pairs[:, 0]] > score[pairs[:, 1]]).mean() > 0.9


def test_policy_from_rewards(dp):
    """A tree policy over four actions, improved from sampled actions and their rewards."""
    rows, actions = 6000, 4
    x, rng = table(rows, 5, 2)
    best = ((x[:, 0] > 0).int() * 2 + (x[:, 1] > 0).int())
    d = dp.DMatrix.from_torch(x)
    model = dp.Booster({"objective": "multi:softprob", "num_class": actions, "max_depth": 3, "eta": 0.5}, [d])
    gen = torch.Generator("cuda").manual_seed(0)
    start, rewards, step = model.train_margin(d), [], 0
    for _ in range(8):
        margin = model.train_margin(d)
        action = torch.multinomial(torch.softmax(margin, 1), 1, generator=gen)[:, 0].int()
        reward = (action == best).float()
        rewards.append(reward.mean().item())
        old, _ = dp.log_prob(margin, action)
        ref, _ = dp.log_prob(start, action)
        for _ in range(3):
            r = dp.policy_loss(model.train_margin(d), action, old, reward - reward.mean(), ref_log_prob=ref, kl=0.01,
                               hess=True)
            model.boost(d, step, r.grad, r.hess)
            step += 1
    assert abs(rewards[0] - 0.25) < 0.05 and rewards[-1] > 0.6
