"""The example's book of sequences and pages (examples/attention_block.py) on the host: a call that finds no room, or is
asked for a sequence that has been started, leaves everything as it was."""
import importlib.util
from pathlib import Path

import pytest

EXAMPLE = Path(__file__).resolve().parents[1] / "xiaomi-hexagon-exl3_amd" / "examples" / "attention_block.py"


@pytest.fixture
def block():
    spec = importlib.util.spec_from_file_location("attention_block_host", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    b = object.__new__(mod.AttentionBlock)
    b.cache, b.free, b.owned, b.length = dict(bits=4, page_tokens=16), [4, 3, 2, 1, 0], {}, {}
    return b


def state(b):
    return list(b.free), {s: list(p) for s, p in b.owned.items()}, dict(b.length)


def test_prompt_without_room_takes_nothing(block):
    before = state(block)
    with pytest.raises(RuntimeError, match="no free page"):
        block.prompt(None, [0, 1], [33, 49])  # three pages and four, of five
    assert state(block) == before
    with pytest.raises(RuntimeError, match="no free page"):
        block.prompt(None, [0], [81])
    assert state(block) == before


def test_prompt_of_a_started_sequence_takes_nothing(block):
    block.owned, block.length, block.free = {7: [0]}, {7: 3}, [4, 3, 2, 1]
    before = state(block)
    for seqs in ([1, 7], [2, 2]):
        with pytest.raises(ValueError):
            block.prompt(None, seqs, [5, 5])
        assert state(block) == before


def test_plan_without_room_takes_nothing(block):
    block.owned, block.length, block.free = {0: [0], 1: [1, 2]}, {0: 16, 1: 32}, [3]
    before = state(block)
    with pytest.raises(RuntimeError, match="no free page"):
        block.plan([0, 1])
    assert state(block) == before
    with pytest.raises(ValueError):
        block.plan([0, 0])
    assert state(block) == before
