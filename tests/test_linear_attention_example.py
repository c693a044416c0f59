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
