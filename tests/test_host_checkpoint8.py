"""checkpoint8 without a GPU: its bookkeeping around the module (what it keeps, draws and differentiates), with
exact copies in the place of the two device calls, so that a checkpointed module's results are the plain
module's, bit for bit."""
import importlib

import pytest
import torch
from torch import nn

from morphocore_amd.functional import Packed8, checkpoint8


@pytest.fixture(autouse=True)
def exact_copies(monkeypatch):
    module = importlib.import_module("morphocore_amd.functional.checkpoint8")
    monkeypatch.setattr(module, "pack8", lambda x: Packed8(x.detach().clone(), torch.zeros(1)))
    monkeypatch.setattr(module, "unpack8", lambda packed, dtype: packed.codes.to(dtype, copy=True))


def both(module, make_input, use=lambda out, x: out):
    """Output and gradients (of the parameters, and of the input where it has one) with and without the checkpoint;
    `use` makes the result from the output and the input as the module left it."""
    results = []
    for call in (module, lambda x: checkpoint8(module, x)):
        torch.manual_seed(5)
        leaf, x = make_input()
        y = use(call(x), x)
        wanted = [p for p in module.parameters() if p.requires_grad] + [leaf] * leaf.requires_grad
        grads = torch.autograd.grad(y, wanted, torch.linspace(-1, 2, y.numel()).view(y.shape), allow_unused=True)
        results.append([y, x.detach(), *grads])
    for plain, kept in zip(*results):
        assert (plain is None and kept is None) or torch.equal(plain, kept)


def leaf_without_gradient():
    x = torch.randn(4, 6)
    return x, x


def inner_with_gradient():
    leaf = torch.randn(4, 6, requires_grad=True)
    return leaf, leaf * 1.5


class ScaleInPlace(nn.Module):
    def __init__(self):
        super().__init__()
        self.scale = nn.Parameter(torch.linspace(0.5, 2, 6))

    def forward(self, x):
        return x.mul_(self.scale)


IN_PLACE = [lambda: nn.Sequential(nn.LeakyReLU(0.1, inplace=True), nn.Linear(6, 3)), lambda: nn.Sequential(nn.LeakyReLU(0.1, inplace=True)),
            lambda: nn.Sequential(nn.LeakyReLU(0.1, inplace=True), nn.Flatten(0)), ScaleInPlace,
            lambda: nn.Sequential(nn.Linear(6, 6), nn.LeakyReLU(0.1, inplace=True))]


@pytest.mark.parametrize("make", IN_PLACE)
def test_module_that_writes_to_its_input(make):
    """The gradients are those at the values that the module was given, not those that it left."""
    torch.manual_seed(0)
    module = make()
    if any(True for _ in module.parameters()):
        both(module, leaf_without_gradient)
    both(module, inner_with_gradient)


@pytest.mark.parametrize("make", IN_PLACE)
def test_input_used_after_the_module_wrote_to_it(make):
    torch.manual_seed(0)
    both(make(), inner_with_gradient, lambda out, x: out.sum() + (x * x).sum())
    both(make(), inner_with_gradient, lambda out, x: (x * x).sum() + 0 * out.sum().detach())


def test_leaf_that_needs_a_gradient_is_not_written_to():
    """As without the checkpoint."""
    x = torch.randn(4, 6, requires_grad=True)
    for call in (lambda m: m(x), lambda m: checkpoint8(m, x)):
        with pytest.raises(RuntimeError, match="leaf Variable that requires grad"):
            call(nn.Sequential(nn.LeakyReLU(0.1, inplace=True), nn.Linear(6, 3)))


class Noise(nn.Module):
    """Draws whatever its training flag."""

    def forward(self, x):
        return x * torch.rand(x.shape) + x * torch.rand(x.shape).sqrt()


def part_in_training(module):
    """A container in evaluation whose dropout is in training."""
    module.eval()
    module[1].train()
    return module


DRAWING = [lambda: nn.Sequential(nn.Linear(6, 6), nn.Dropout(0.5)), lambda: nn.Sequential(nn.Linear(6, 6), nn.Dropout(0.5)).eval(),
           lambda: part_in_training(nn.Sequential(nn.Linear(6, 6), nn.Dropout(0.5))), lambda: nn.Sequential(nn.Linear(6, 6), Noise()),
           lambda: nn.Sequential(nn.Linear(6, 6), Noise()).eval(), lambda: nn.Sequential(nn.Dropout(0.5, inplace=True), nn.Linear(6, 3))]


@pytest.mark.parametrize("make", DRAWING)
def test_rerun_draws_the_forwards_numbers(make):
    torch.manual_seed(0)
    module = make()
    both(module, inner_with_gradient)
    both(module, leaf_without_gradient)
    # The caller's generator goes on as if the module had run once.
    x = torch.randn(4, 6)
    torch.manual_seed(7)
    module(x.clone())
    want = torch.rand(3)
    torch.manual_seed(7)
    out = checkpoint8(module, x.clone())
    torch.autograd.grad(out.sum(), module.parameters())
    assert torch.equal(torch.rand(3), want)


def test_states_that_are_not_kept():
    """preserve_rng=False: the rerun draws on from the generator as it is."""
    module, x = nn.Sequential(nn.Linear(6, 6), nn.Dropout(0.5)), torch.randn(40, 6)
    torch.manual_seed(7)
    out = checkpoint8(module, x, preserve_rng=False)
    got = torch.autograd.grad(out.sum(), module[0].bias)[0]
    torch.manual_seed(7)
    module(x)
    want = torch.autograd.grad(module(x).sum(), module[0].bias)[0]
    assert torch.equal(got, want)
    from morphocore_amd.nn import Checkpoint8
    assert Checkpoint8(module).preserve_rng and not Checkpoint8(module, preserve_rng=False).preserve_rng
