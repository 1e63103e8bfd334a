"""The example that trains on choices: every loss does what it is for."""
import pathlib
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")


def test_learn_from_choices():
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))
    import learn_from_choices as example
    out = example.main(["--rows", "6000", "--rounds", "24"])
    first, last = out["rank"]
    assert abs(first - 0.6931) < 1e-3 and last < 0.3
    first, last = out["episodes"]
    assert abs(first - 0.25) < 1e-3 and last > 0.3
    first, last = out["policy"]
    assert abs(first - 0.25) < 0.05 and last > 0.6
