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
