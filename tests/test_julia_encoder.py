"""CPU checks of the Julia extension's encoder drivers, without Julia: their conditions on sizes, read from the
source, against those of the Python layer."""
import re

import pytest

from test_julia_token_block import body


def condition(function, refused):
    """The Julia expression before `|| throw(DimensionMismatch(refused))`, as Python."""
    text = re.search(rf"^\s*([^\n]*?)\s*\|\|\s*throw\(DimensionMismatch\(\"{refused}\"\)\)", body(function), re.M).group(1)
    return text.replace("&&", " and ").replace("||", " or ")


@pytest.mark.parametrize("heads,kv_heads,good", [
    (0, 0, True), (4, 4, True), (8, 2, True), (3, 2, False), (2, 4, False), (0, 2, False), (2, 0, False)])
def test_heads_that_share(heads, kv_heads, good):
    """Key heads that no query head shares are refused: their gradients would be nobody's."""
    said = eval(condition("attention_sizes", "heads"), {}, {"heads": heads, "kv_heads": kv_heads})  # noqa: S307
    assert bool(said) == good


def test_what_is_kept_has_the_header_s_size():
    """A float a query row and head, whatever the batch."""
    text = body("attention")
    assert re.search(r"top = keep \? similar\(q, Float32, size\(q\)\[2:end\]\) : nothing", text)
    assert re.search(r"length\(top\) == length\(q\) ÷ max\(dim, 1\) \|\| throw", body("attention_pullback"))
