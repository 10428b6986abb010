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
