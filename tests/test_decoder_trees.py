"""Which trees a leaf decoder takes for one another's, and what it does with the gradients (on the CPU, up to the first operator)."""
import copy

import pytest
import torch

import svox_amd as svox


def pair(**kw):
    features = svox.N3Tree(data_format=None, data_dim=12, init_refine=1, **kw)
    tree = svox.N3Tree(data_format="SH1", init_refine=1, **kw)
    return features, tree, svox.LeafDecoder(12, tree.data_dim, hidden=40)


def taken(decoder, features, tree):
    """Whether the trees are taken for one structure: the first operator then refuses tensors that are not on a GPU."""
    with pytest.raises((ValueError, RuntimeError)) as e:
        decoder.decode_tree(features, tree)
    assert "same structure" in str(e.value) or "CUDA tensor" in str(e.value), e.value
    return "CUDA tensor" in str(e.value)


def cell(node, x, y, z):
    return tuple(torch.tensor([v]) for v in (node, x, y, z))


def test_trees_divided_at_different_cells_are_refused():
    features, tree, decoder = pair(init_reserve=5)
    assert features.capacity == tree.capacity and taken(decoder, features, tree)
    features.refine(sel=cell(1, 0, 0, 0))
    assert features.capacity == tree.capacity and not taken(decoder, features, tree)
    tree.refine(sel=cell(1, 1, 0, 1))       # as many nodes, another cell
    assert features.n_internal == tree.n_internal and not taken(decoder, features, tree)
    features.refine(sel=cell(1, 1, 0, 1))
    tree.refine(sel=cell(1, 0, 0, 0))       # the same cells, in another order: the records lie elsewhere
    assert features.n_leaves == tree.n_leaves and not taken(decoder, features, tree)


def test_spare_capacity_makes_no_difference():
    features, tree, decoder = pair()
    roomy = svox.N3Tree(data_format="SH1", init_refine=1, init_reserve=7)
    assert roomy.capacity > features.capacity and taken(decoder, features, roomy)
    for t in (features, roomy):
        t.refine(sel=cell(2, 0, 1, 0))
    assert taken(decoder, features, roomy) and not taken(decoder, features, tree)


def test_what_is_known_of_two_trees_goes_with_their_structure():
    features, tree, decoder = pair(init_reserve=5)
    third = svox.N3Tree(data_format="SH1", init_refine=1)
    assert taken(decoder, features, tree) and taken(decoder, features, tree) and taken(decoder, features, third)
    assert features._structure() is tree._structure()
    tree.data.data += 1
    assert features._structure() is tree._structure()
    tree.child[3, 0, 0, 0] = 1              # (a torch operation on the table itself)
    assert not taken(decoder, features, tree) and taken(decoder, features, third)
    tree.child[3, 0, 0, 0] = 0
    assert taken(decoder, features, tree)
    for t in (features, tree):
        t.refine()
        t.merge()
    assert taken(decoder, features, tree) and not taken(decoder, features, third)
    tree.shrink_to_fit()
    assert not taken(decoder, features, tree)
    features.shrink_to_fit()
    assert taken(decoder, features, tree) and taken(decoder, *copy.deepcopy((features, tree)))
    loaded = svox.N3Tree(data_format="SH1", init_refine=2)
    loaded.load_state_dict(svox.N3Tree(data_format="SH1", init_refine=2).state_dict())
    assert not taken(decoder, features, loaded)


def test_other_branching_factors_are_refused():
    features, tree, decoder = pair()
    assert not taken(decoder, features, svox.N3Tree(N=3, data_format="SH1"))
    assert not taken(decoder, svox.N3Tree(N=3, data_format=None, data_dim=12), svox.N3Tree(data_format="SH1"))


class Plain(svox.LeafDecoder):
    """A decoder whose network is one product, of torch's own."""

    def forward(self, x):
        return x @ self.ffns[0].w_gate.t()


def plain():
    features, tree, _ = pair()
    torch.manual_seed(0)
    features.data.data.normal_()
    return features, tree, Plain(12, tree.data_dim, hidden=tree.data_dim)


def test_a_loss_without_the_records():
    features, tree, decoder = plain()
    other = torch.ones(3, requires_grad=True)
    assert decoder.backward_through(features, tree, lambda: (other ** 2).sum()) == 3
    assert torch.equal(other.grad, torch.full((3,), 2.0)) and features.data.grad is None and decoder.ffns[0].w_gate.grad is None


def test_a_tree_that_requires_no_gradient_is_refused_before_anything_is_done():
    features, tree, decoder = plain()
    tree.data.requires_grad_(False)
    other = torch.ones(3, requires_grad=True)
    with pytest.raises(ValueError, match="does not require a gradient"):
        decoder.backward_through(features, tree, lambda: (other ** 2).sum() + tree.data.sum())
    assert other.grad is None and not bool(tree.data.any())


def test_records_that_are_computed_from_something_else_are_refused():
    features, tree, decoder = plain()
    torch.nn.utils.parametrize.register_parametrization(tree, "data", torch.nn.Softplus())
    with pytest.raises(ValueError, match="computed from something else"):
        decoder.backward_through(features, tree, lambda: (tree.data ** 2).sum())


def test_gradients_add_up_and_nothing_trained_is_no_error():
    features, tree, decoder = plain()
    loss = lambda: (tree.data ** 2).sum()  # noqa: E731
    decoder.backward_through(features, tree, loss)
    once = decoder.ffns[0].w_gate.grad.clone(), features.data.grad.clone()
    x, w = features.data.detach().reshape(-1, 12), decoder.ffns[0].w_gate.detach()
    records = x @ w.t()
    torch.testing.assert_close(once[0], 2 * records.t() @ x)
    torch.testing.assert_close(once[1].reshape(-1, 12), 2 * records @ w)
    decoder.backward_through(features, tree, loss)
    torch.testing.assert_close(decoder.ffns[0].w_gate.grad, 2 * once[0])
    decoder.requires_grad_(False)
    features.data.requires_grad_(False)
    assert decoder.backward_through(features, tree, loss) == loss().detach()


def test_the_gradient_a_tree_holds_stays():
    features, tree, decoder = plain()
    held = torch.randn_like(tree.data)
    tree.data.grad = held.clone()
    decoder.backward_through(features, tree, lambda: (tree.data ** 2).sum())
    want = decoder.ffns[0].w_gate.grad.clone()
    assert torch.equal(tree.data.grad, held)
    decoder.zero_grad()
    tree.data.grad = None
    decoder.backward_through(features, tree, lambda: (tree.data ** 2).sum())
    assert tree.data.grad is None and torch.equal(decoder.ffns[0].w_gate.grad, want)

    def fails():
        (tree.data ** 2).sum().backward()
        raise KeyError("no rays")

    tree.data.grad = held.clone()
    with pytest.raises(KeyError):
        decoder.backward_through(features, tree, fails)
    assert torch.equal(tree.data.grad, held)


def test_trees_made_in_inference_mode():
    with torch.inference_mode():
        features, tree, decoder = pair(init_reserve=5)
        assert taken(decoder, features, tree) and taken(decoder, features, tree)
        features.child[1, 0, 0, 0] = 1
        assert not taken(decoder, features, tree)
