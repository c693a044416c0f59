"""The example's book of sequences and states (examples/linear_attention_block.py) on the host: a call that finds no
free state leaves everything as it was."""
import importlib.util
from pathlib import Path

import pytest

EXAMPLE = Path(__file__).resolve().parents[1] / "xiaomi-hexagon-exl3_amd" / "examples" / "linear_attention_block.py"


@pytest.fixture
def block():
    spec = importlib.util.spec_from_file_location("linear_attention_block_host", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    b = object.__new__(mod.LinearAttentionBlock)
    b.free, b.slot = [2, 1, 0], {}
    return b


def test_sequences_take_and_free_states(block):
    assert block._take(["a", "b"]) == ([-1, -1], [0, 1])
    assert block._take(["b", "c"]) == ([1, -1], [1, 2])
    with pytest.raises(RuntimeError, match="no free state"):
        block._take(["a", "d"])
    assert (block.free, block.slot) == ([], {"a": 0, "b": 1, "c": 2})
    block.release("b")
    block.release("unknown")
    assert block._take(["d"]) == ([-1], [1])


def test_a_sequence_named_twice_takes_nothing(block):
    with pytest.raises(ValueError, match="twice"):
        block.rows(None, None, ["a", "a"], [1, 1])
    with pytest.raises(RuntimeError, match="no free state"):
        block.rows(None, None, list("abcd"), [1] * 4)
    assert (block.free, block.slot) == ([2, 1, 0], {})


def test_a_call_that_fails_takes_nothing(block):
    """a new sequence whose rows() failed would go on from whatever its slot held"""
    torch = pytest.importorskip("torch")
    assert block._take(["old"]) == ([-1], [0])
    x = torch.zeros(3, 8)
    for seqs, lens in ((["a"], [2]), (["a"], [4]), (["a", "b"], [3]), (["a"], [1, 2]), (["a", "b"], [4, -1]), ([], [3])):
        with pytest.raises(ValueError, match="lengths"):
            block.rows(x, x, seqs, lens)
        assert (block.free, block.slot) == ([2, 1], {"old": 0}), (seqs, lens)

    def fails(*_):
        raise RuntimeError("refused")

    block._block, block.workspace, block.max_rows = fails, None, 32
    with pytest.raises(Exception):
        block.rows(x, x, ["old", "a", "b"], [1, 1, 1])
    assert (block.free, block.slot) == ([2, 1], {"old": 0})


def test_a_plan_names_a_sequence_once(block):
    """two sequences in one slot would race for its state"""
    block._take(["a", "b"])
    with pytest.raises(ValueError, match="twice"):
        block.plan(["a", "b", "a"])
    with pytest.raises(KeyError):
        block.plan(["c"])
