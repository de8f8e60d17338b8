"""CPU checks of the Julia extension's token-block drivers, without Julia: what `similar` makes and no
kernel writes has to be written by the driver."""
import re

from test_julia_ext import EXT


def body(name):
    text = re.sub(r"#[^\n]*", "", open(EXT).read())
    return re.search(rf"^function {name}\(.*?^end$", text, re.M | re.S).group(0)


def test_gate_gradient_of_no_rows_is_zero():
    """fms_block_norm_pullback writes one gate vector for gate_rows rows: with no rows none, though a
    shared gate has one."""
    pullback = body("block_norm_pullback")
    assert re.search(r"dgate\b.*=.*like\(gate\)", pullback)  # (uninitialised)
    assert re.search(r"^\s*rows == 0 && dgate !== nothing && fill!\(dgate, 0\)\s*$", pullback, re.M)
