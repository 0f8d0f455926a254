"""The policy-gradient example: the parameters' first plane after a step is the derivative of the trained
weights by the entropy bonus.  One step is linear in the bonus, so that derivative is the difference of
two steps whose bonuses are 1 apart."""

import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("policy_step", ROOT / "examples" / "policy_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_first_plane_is_the_derivative_by_the_bonus(example):
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 96, (2, 33), generator=g).cuda()
    advantage = torch.randn(2, 32, generator=g).cuda()

    def after(bonus):
        model = example.Decoder(vocab=96, width=128, heads=2, layers=2, degree=1, positions=40)
        loss = example.policy_step(model, ids, advantage, bonus=bonus, dropout=0.25, seed=3)
        return model, loss

    (near, loss), (far, _) = after(0.01), after(1.01)
    start = example.Decoder(vocab=96, width=128, heads=2, layers=2, degree=1, positions=40)
    assert len(loss) == 2 and loss[1] < 0     # d loss / d bonus = -entropy
    for name, w in near.p.items():
        moved = far.p[name].coeffs[0].double() - near.p[name].coeffs[0].double()
        got = w.coeffs[1].double()
        # float32 weights of size w: their difference carries 2^-23 |w| of rounding; a gradient through a
        # few float32 products (2^-16 each) carries 2^-14 of its size, in both runs, of which the part that
        # the bonus does not enter is the step taken with almost none
        step = (w.coeffs[0].double() - start.p[name].coeffs[0].double()).norm()
        room = 2.0 ** -22 * w.coeffs[0].double().norm() + 2.0 ** -12 * got.norm() + 2.0 ** -13 * step
        assert (got - moved).norm() <= room, name


def test_next_tokens(example):
    model = example.Decoder(vocab=96, width=128, heads=2, layers=1, degree=1, positions=40)
    ids = torch.randint(0, 96, (3, 7), generator=torch.Generator().manual_seed(6)).cuda()
    tokens, log_probs = example.next_tokens(model, ids, top=4)
    with example.PolyTensor.plain_range(), torch.no_grad():
        want = torch.log_softmax(model.logits(ids)[:, -1].value.double(), -1)
    best = torch.sort(want, descending=True, stable=True)
    assert torch.equal(tokens, best.indices[:, :4])
    torch.testing.assert_close(log_probs.double(), best.values[:, :4], rtol=1e-5, atol=1e-5)
