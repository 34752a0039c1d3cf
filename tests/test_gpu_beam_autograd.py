"""beam_reorder writes its states in place and has no gradient: autograd must see the write or refuse it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def dev():
    import nn_amd
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nn_amd.init(0)
    return torch.device("cuda:0")


def cache(seed=0):
    return torch.randn(6, 2, 9, 8, generator=torch.Generator().manual_seed(seed)).cuda()


PARENTS = [[1, 1, 0], [2, 0, 2]]
ROWS = [1, 1, 0, 5, 3, 5]


def test_a_backward_pass_over_a_moved_state_raises():
    import nn_amd
    parents = torch.tensor(PARENTS, device="cuda")
    for view in (lambda c: c, lambda c: c[:, :, :4]):
        c, w = cache(), torch.ones(8, device="cuda", requires_grad=True)
        y = (c * w).sum()  # c is saved for w's gradient
        nn_amd.beam_reorder([view(c)], parents)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    c, w = cache(), torch.ones(8, device="cuda", requires_grad=True)
    nn_amd.beam_reorder(c, parents)  # before it is used
    (c * w).sum().backward()
    ref = cache()[ROWS]
    assert torch.equal(c, ref)
    assert torch.equal(w.grad, torch.autograd.grad((ref * w).sum(), w)[0])


def test_a_state_that_requires_grad_is_refused_before_any_moves():
    import nn_amd
    parents = torch.tensor(PARENTS, device="cuda")
    a, b = cache(1), cache(2).requires_grad_()
    for states in ([a, b], [a, b * 2.0], b):
        with pytest.raises(nn_amd.Unsupported, match="no_grad"):
            nn_amd.beam_reorder(states, parents)
    assert torch.equal(a, cache(1)) and torch.equal(b, cache(2))
    with torch.no_grad():
        nn_amd.beam_reorder([a, b], parents)
    assert torch.equal(a, cache(1)[ROWS]) and torch.equal(b.detach(), cache(2)[ROWS]) and b.requires_grad


def test_states_of_inference_mode_and_empty_lists():
    import nn_amd
    parents = torch.tensor(PARENTS, device="cuda")
    with torch.inference_mode():
        c = cache(3)
        nn_amd.beam_reorder([c[:, :, :5], c[:, :, 5:]], parents)
    assert torch.equal(c, cache(3)[ROWS])
    nn_amd.beam_reorder([c], parents)  # and of such a tensor outside
    assert torch.equal(c, cache(3)[ROWS][ROWS])
    nn_amd.beam_reorder([], parents)
    nn_amd.beam_reorder(torch.empty(6, 0, device="cuda"), parents)
