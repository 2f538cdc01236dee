"""Dropout's passes and stacks of blocks on the CPU, by the definition in the kernels' place."""
import copy
import io

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import matrix_linear, packed4, residual

import packed4_oracle as po
import residual_oracle as ro


def _kept(shape, drop):
    seed, offset = (int(v) for v in drop.seed) if isinstance(drop.seed, torch.Tensor) else (drop.seed, drop.offset)
    return ro.mask(tuple(shape), drop.p, seed, offset, drop.per)


@pytest.fixture
def definition(monkeypatch):
    """dropout, norm and join by their formulas, with torch's own gradients."""
    def dropout(x, drop, axis=-1):
        kept, scale = _kept(x.shape, drop)
        return torch.where(kept, x * scale, torch.zeros_like(x))

    def norm(x, n, axis=-1):
        return ro.norm(x, n.kind, n.weight, n.bias, n.eps)

    def join(f, x, post, gate, pre, drop, a, b, axis=-1):
        v = f if post is None else norm(f, post)
        v = v if drop is None else dropout(v, drop)
        s = a * x + b * (v if gate is None else v * gate)
        return s, norm(s, pre)
    for name, f in (("dropout", dropout), ("norm", norm), ("join", join)):
        monkeypatch.setattr(residual, name, f)


def _modules(counter):
    return [pkg.Dropout(0.4, seed=5 + i, counter=counter) for i in range(2)]


@pytest.mark.parametrize("counter", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_passes_that_are_run_again(definition, counter, reentrant):
    """The mask of the gradient is that of the result, with several passes on their way, whichever goes back first; masks are those of passes that are not run again."""
    for order in ((0, 1, 2), (2, 1, 0), (1, 2, 0)):
        ms, plain = _modules(counter), _modules(counter)
        leaves = [(torch.randn(6, 24) + 3).requires_grad_() for _ in order]
        run = lambda x: ms[1](torch.sin(ms[0](x * 1.5)))  # noqa: E731,B023
        ys = [checkpoint(run, x, use_reentrant=reentrant) for x in leaves]
        want = [plain[1](torch.sin(plain[0](x * 1.5))) for x in leaves]
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
        for i in order:
            (a,), (b,) = (torch.autograd.grad(y[i].sum(), leaves[i]) if not reentrant else (_through(y[i], leaves[i]),) for y in (ys, want))
            assert torch.equal(a, b)
        # a run again is no pass of its own
        assert [int(m.state[1]) if counter else m.calls for m in ms] == [3, 3]
        assert torch.equal(ms[0](leaves[0]), plain[0](leaves[0]))


def _through(y, leaf):
    leaf.grad = None
    y.sum().backward()
    return leaf.grad


@pytest.mark.parametrize("counter", [False, True])
def test_nested_and_twice(definition, counter):
    ms, plain = _modules(counter), _modules(counter)
    x = (torch.randn(5, 16) + 3).requires_grad_()
    inner = lambda v: ms[0](v).exp()  # noqa: E731
    y = checkpoint(lambda v: ms[1](checkpoint(inner, v.sin(), use_reentrant=False)).cos(), x, use_reentrant=False)
    want = plain[1](plain[0](x.sin()).exp()).cos()
    (b,) = torch.autograd.grad(want.sum(), x)
    for _ in range(2):
        (a,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
        assert torch.equal(a, b)
    # one module twice in a pass
    y = checkpoint(lambda v: ms[0](ms[0](v).exp()).sin(), x, use_reentrant=False)
    want = plain[0](plain[0](x).exp()).sin()
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(want.sum(), x)[0])


@pytest.mark.parametrize("counter", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_stacks(definition, counter, reentrant):
    def make():
        torch.manual_seed(7)
        return pkg.ResidualStack([torch.nn.Sequential(torch.nn.Linear(24, 40), torch.nn.SiLU(), torch.nn.Linear(40, 24)) for _ in range(3)], 24, post=True, gate=0.5, drop=0.4,
                                 per="element", counter=counter)
    stack, plain = make(), make()
    for _ in range(2):
        x = torch.randn(4, 9, 24).requires_grad_()
        y, want = checkpoint(stack, x, use_reentrant=reentrant), plain(x)
        assert torch.equal(y, want)
        y.square().sum().backward()
        got = [x.grad] + [p.grad for p in stack.parameters()]
        x.grad = None
        want.square().sum().backward()
        for a, b in zip(got, [x.grad] + [p.grad for p in plain.parameters()]):
            # (gradients of several uses are added up in another order)
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())


@pytest.mark.parametrize("counter", [False, True])
def test_runs_again_that_cannot_be_told(definition, counter):
    """Refused, not given another mask."""
    m = pkg.Dropout(0.4, counter=counter)
    x = torch.randn(6, 24).requires_grad_()
    run = lambda v: m(v.sin()).exp()  # noqa: E731
    for reentrant in (False, True):
        y = checkpoint(run, x, use_reentrant=reentrant, preserve_rng_state=False)
        with pytest.raises(RuntimeError, match="run again in a backward pass"):
            y.sum().backward()
    # two passes from the same state of torch's generator: one after the other, and both on their way
    for _ in range(3):
        torch.manual_seed(1)
        y = checkpoint(run, x, use_reentrant=False)
        (g,) = torch.autograd.grad(y.sum(), x)
        assert torch.equal(g != 0, y != 1)
    torch.manual_seed(2)
    first = checkpoint(run, x, use_reentrant=False)
    torch.manual_seed(2)
    second = checkpoint(run, x, use_reentrant=False)
    for y in (first, second):
        with pytest.raises(RuntimeError, match="run again in a backward pass"):
            y.sum().backward()
    # a pass whose number is kept no longer
    y = checkpoint(run, x, use_reentrant=False)
    with torch.no_grad():
        for _ in range(residual.PASSES_KEPT):
            m.draw()
    with pytest.raises(RuntimeError, match="run again in a backward pass"):
        y.sum().backward()


def test_other_passes_leave_the_generator_alone(definition):
    m = pkg.Dropout(0.4, seed=1)
    before = torch.get_rng_state()
    y = m(torch.randn(3, 8, generator=torch.Generator()).requires_grad_())
    y.sum().backward()
    m.eval()
    with torch.no_grad():
        m(torch.ones(3, 8))
    assert torch.equal(torch.get_rng_state(), before)
    assert not m._passes


def test_what_is_kept_of_passes_stays_here(definition):
    m = pkg.Dropout(0.4, seed=1, counter=True)
    with torch.no_grad():
        m(torch.ones(3, 8))
    assert len(m._passes) == 1
    buffer = io.BytesIO()
    torch.save(m, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(m), torch.load(buffer, weights_only=False)):
        assert not other._passes and torch.equal(other.state, m.state)
    assert set(m.state_dict()) == set(pkg.Dropout(0.1, counter=True).state_dict())


@pytest.fixture
def pack_on_cpu(monkeypatch):
    monkeypatch.setattr(matrix_linear, "pack4", lambda w: packed4.Packed4.from_parts(*po.pack(w.detach()), w.shape[1], w.dtype))


def test_every_layer_of_a_stack_is_packed(pack_on_cpu):
    """A block that is a layer itself, layers at any depth, and one layer in several places, which stays one."""
    shared, deep = pkg.MatrixLinear(40, 40), pkg.MatrixLinear(40, 40)
    once, pair = pkg.MatrixLinear(40, 40), torch.nn.Sequential(shared, torch.nn.SiLU(), shared)
    blocks = [once, residual.matrix_block(40, 64), pair, shared, once, torch.nn.Sequential(torch.nn.Sequential(deep), torch.nn.Linear(40, 40)), pair]
    for x4 in (False, True):
        stack = pkg.ResidualStack(copy.deepcopy(blocks), 40)
        made = stack.pack4(x4)
        assert made is stack and not any(isinstance(m, pkg.MatrixLinear) for m in stack.modules())
        packed = [m for m in stack.modules() if isinstance(m, pkg.MatrixLinear4)]
        assert len(packed) == 5 and all(m.x4 == x4 for m in packed)
        b = stack.blocks
        assert b[0] is b[4] and b[2] is b[6] and b[2][0] is b[2][2] is b[3] and b[3] is not b[0] and isinstance(b[5][1], torch.nn.Linear)
        for i, layer in ((0, once), (3, shared)):
            assert torch.equal(b[i].weight.parts()[0], po.pack(layer.weight.detach())[0])


@pytest.mark.parametrize("counter", [False, True])
def test_copies_draw_their_own_masks(definition, counter):
    """Unless a seed was given; a state dict, and a module saved whole, go on with the masks of the module that they are from."""
    torch.manual_seed(0)
    x = torch.ones(50, 64)
    m = pkg.Dropout(0.5, counter=counter)
    m(x)
    copies = [copy.deepcopy(m) for _ in range(2)]
    buffer = io.BytesIO()
    torch.save(m, buffer)
    buffer.seek(0)
    whole, loaded = torch.load(buffer, weights_only=False), pkg.Dropout(0.5, counter=counter)
    loaded.load_state_dict(m.state_dict())
    state = [copy.deepcopy(c.state_dict()) for c in copies]
    masks = [v(x) != 0 for v in [m] + copies]
    # (of 3200 values in halves, kept in both: 800, six deviations of 24.5)
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs(int((masks[a] & masks[b]).sum()) - 800) < 147
    assert torch.equal(whole(x) != 0, masks[0]) and torch.equal(loaded(x) != 0, masks[0])
    for c, mask in zip(state, masks[1:]):
        again = pkg.Dropout(0.5, counter=counter)
        again.load_state_dict(c)
        assert torch.equal(again(x) != 0, mask)
    # copies of copies, and one of the copies by itself in a larger module
    layers = copy.deepcopy(torch.nn.ModuleList([copies[0]] * 2 + [copies[1]]))
    assert layers[0] is layers[1] and not torch.equal(layers[0](x), layers[2](x))
    given = pkg.Dropout(0.5, seed=9, counter=counter)
    assert torch.equal(copy.deepcopy(given)(x), given(x))
