"""Which calls a capture refuses, because their backward would come to what was recorded on the default stream: what they ask, without a capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def side():
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        yield
    torch.cuda.current_stream().wait_stream(stream)


MADE = {"view": lambda t: t.view(-1), "cast": lambda t: t.double(), "result": lambda t: (t.relu() * 3).sum(0), "in place": lambda t: t.clone().mul_(2)}


@pytest.mark.parametrize("made", MADE)
def test_tensors_behind_a_leaf(made, side):
    """What is made elsewhere of a leaf that a graph of the default stream holds leads there as the leaf does; and not once that graph is gone."""
    from dfa3D import _lib
    held = _lib.binding().held
    leaf = torch.randn(6, 4, device="cuda", requires_grad=True)
    assert not held(MADE[made](leaf))
    with torch.cuda.stream(torch.cuda.default_stream()):
        eager = leaf * 2
    assert held(leaf) and held(MADE[made](leaf)) and held(eager) and held(MADE[made](eager))
    assert not held(MADE[made](leaf.detach())) and not held(leaf.detach())
    del eager
    assert not held(leaf) and not held(MADE[made](leaf))


def test_a_leaf_behind_many_others(side):
    from dfa3D import _lib
    held = _lib.binding().held
    leaf, other = torch.ones(4, device="cuda", requires_grad=True), torch.ones(4, device="cuda", requires_grad=True)
    with torch.cuda.stream(torch.cuda.default_stream()):
        eager = leaf * 2
    t = other * 1
    for _ in range(40):                                          # (2^40 ways through it)
        t = t + t * 0.5
    assert not held(t) and held(t + leaf)
    del eager


def _dropout():
    from dfa3D.dropout import dropout
    x, r = (torch.randn(6, 8, device="cuda", requires_grad=True) for _ in range(2))
    return (lambda: dropout(x.t(), 0.3, 5, residual=r.t())), 2


def _embedding():
    from dfa3D.embedding import scaled_embedding
    table, scale, plus = (torch.randn(s, device="cuda", requires_grad=True) for s in ((5, 2, 8), (7, 2), (8, 7)))
    index = torch.randint(0, 5, (7,), device="cuda")
    return (lambda: scaled_embedding(table, index, scale=scale, plus=plus.t())), 3


def _norm():
    from dfa3D.norm import level_group_norm
    x, w, b = (torch.randn(s, device="cuda", requires_grad=True) for s in ((2, 8, 5), (8,), (8,)))
    return (lambda: level_group_norm(x.transpose(1, 2), 4, w, b)), 3


@pytest.mark.parametrize("make", [_dropout, _embedding, _norm])
def test_calls_step_by_step_ask_as_well(make, monkeypatch):
    from dfa3D import _lib
    call, operands = make()
    asked = []
    real = _lib.binding().refuse_capture
    monkeypatch.setattr(_lib.binding(), "refuse_capture", lambda *a: asked.append(a) or real(*a))
    call()
    assert len(asked) == 1 and sum(isinstance(t, torch.Tensor) and t.requires_grad for t in asked[0]) == operands
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
        call()
    assert len(asked) == 2
