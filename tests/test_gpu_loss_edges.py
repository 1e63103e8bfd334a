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
