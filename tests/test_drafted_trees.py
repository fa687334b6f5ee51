"""CPU tests of the drafted-tree helpers of the decoder."""
import pytest

from onnx_runtime_dart_b200 import ArgumentError
from onnx_runtime_dart_b200.decoder import accepted_path, tree_arrays


def test_tree_arrays():
    bits, depth = tree_arrays([-1, 0, 0, 1, 3, 2])
    assert bits == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100101]
    assert depth == [0, 1, 1, 2, 3, 2]
    assert tree_arrays([-1]) == ([1], [0])
    bits, depth = tree_arrays([-1] + list(range(63)))
    assert bits[63] == (1 << 64) - 1 and depth[63] == 63


@pytest.mark.parametrize("parents", [[0], [-1, -1], [-1, 1], [-1, 0, 3, 1], [-1, 2, 0]])
def test_tree_arrays_refuses(parents):
    with pytest.raises(ArgumentError, match="root"):
        tree_arrays(parents)


def test_accepted_path():
    parents, tokens = [-1, 0, 0, 1, 3], [5, 7, 8, 9, 1]
    assert accepted_path(tokens, parents, [7, 9, 0, 1, 4]) == [0, 1, 3, 4]
    assert accepted_path(tokens, parents, [8, 9, 0, 1, 4]) == [0, 2]
    assert accepted_path(tokens, parents, [6, 9, 0, 1, 4]) == [0]
    assert accepted_path([5], [-1], [5]) == [0]
    # two children with the same token: the first counts
    assert accepted_path([1, 2, 2, 3], [-1, 0, 0, 2], [2, 3, 3, 0]) == [0, 1]
