"""Outputs of the choice losses that overlap what a call reads, or each other, are
refused before any device work (no GPU): another thread would read what has
been written over."""
import pytest

BASE = 1 << 20  # addresses that no refused call reads
FAR = 1 << 12   # bytes from one array to the next


def refused(dp, name, *args):
    assert getattr(dp.lib(), name)(*args) == -1
    return dp.lib().XGBGetLastError().decode()


NAMES = ("score", "ref", "weight", "loss", "grad", "hess", "begin")


def preference(dp, **at):
    """dp_preference_loss over 8 rows in 4 pairs, every array apart but for `at`."""
    a = {name: BASE + i * FAR for i, name in enumerate(NAMES)}
    for name, address in at.items():
        a[name] = address
    return refused(dp, "dp_preference_loss", 8, a["begin"], 4, a["score"], a["ref"], a["weight"], 1.0, 0.0, a["loss"],
                   a["grad"], a["hess"], None)


@pytest.mark.parametrize("out", ["loss", "grad", "hess"])
@pytest.mark.parametrize("other", NAMES)
def test_preference_outputs(dp, out, other):
    if out == other:
        pytest.skip("the array itself")
    address = {name: BASE + i * FAR for i, name in enumerate(NAMES)}
    size = {"score": 32, "ref": 32, "weight": 16, "loss": 16, "grad": 32, "hess": 32, "begin": 72}
    for at in (address[other], address[other] + size[other] - 4, address[other] - size[out] + 4):
        assert "overlap" in preference(dp, **{out: at})


ROW_IN = ("label", "old", "ref", "advantage", "weight")


def policy(dp, rows=4, **at):
    """dp_policy_loss over rows of 10 fp32 classes 16 apart, every array apart but for `at`."""
    names = ("margin", "label", "old", "ref", "advantage", "weight", "loss", "log_prob", "grad", "hess")
    a = {name: BASE + i * FAR for i, name in enumerate(names)}
    a.update(at)
    return refused(dp, "dp_policy_loss", 0, a["margin"], rows, 10, 16, a["label"], a["old"], a["ref"], a["advantage"],
                   a["weight"], 0.2, 0.2, 0.1, a["loss"], a["log_prob"], a["grad"], 16, a["hess"], 16, None)


@pytest.mark.parametrize("out", ["loss", "log_prob"])
def test_policy_vectors(dp, out):
    names = ("margin", "label", "old", "ref", "advantage", "weight", "loss", "log_prob", "grad", "hess")
    address = {name: BASE + i * FAR for i, name in enumerate(names)}
    assert "overlaps the margins" in policy(dp, **{out: address["margin"]})
    assert "overlaps the margins" in policy(dp, **{out: address["margin"] + 3 * 64 + 36})
    assert "overlaps the margins" in policy(dp, **{out: address["margin"] + 52})  # from the gap into the next row
    assert "gradient or the curvature" in policy(dp, **{out: address["grad"] + 64})
    assert "gradient or the curvature" in policy(dp, **{out: address["hess"] - 12})
    for other in ROW_IN:
        assert "an output vector overlaps an input vector" in policy(dp, **{out: address[other] + 4})
    assert "two output vectors" in policy(dp, loss=address["log_prob"], log_prob=address["log_prob"])
    for other in ROW_IN:
        assert "the gradient or the curvature overlaps" in policy(dp, **{other: address["grad"] + 128})
        assert "the gradient or the curvature overlaps" in policy(dp, **{other: address["hess"]})


def test_log_prob_vectors(dp):
    lead = lambda margin, label: (0, margin, 4, 10, 16, label)  # noqa: E731
    a = [BASE + i * FAR for i in range(7)]
    call = lambda label=a[1], logp=a[2], norm=a[3]: refused(dp, "dp_log_prob", *lead(a[0], label), logp, norm, None)  # noqa: E731
    assert "margins" in call(logp=a[0] + 64)
    assert "margins" in call(norm=a[0] + 32)
    assert "two output vectors" in call(logp=a[3] + 8)
    assert "input vector" in call(norm=a[1])
    assert "input vector" in call(logp=a[1] + 4)
    grad = lambda label=a[1], norm=a[2], weight=a[3], hess=a[5]: refused(  # noqa: E731
        dp, "dp_log_prob_grad", *lead(a[0], label), norm, weight, a[4], 16, hess, 16, None)
    for name in ("label", "norm", "weight"):
        assert "the gradient or the curvature overlaps" in grad(**{name: a[4] + 64})
        assert "the gradient or the curvature overlaps" in grad(**{name: a[5]})
