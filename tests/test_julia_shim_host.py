"""The Julia shim is not executed here (no Julia); what is checked is its text: each method that hands sizes of
several arrays to the library compares them first, as the Python side does."""
import os
import re

SHIM = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "knet.jl_b200", "julia", "LibKnetSM100.jl")


def method(name):
    text = open(SHIM).read()
    m = re.search(r"^( *)function %s\(.*?^\1end" % re.escape(name), text, re.S | re.M)
    return m.group(0)


def test_linear_nll_compares_sizes_before_the_call():
    """Labels, bias, features or a forward result that are too short would be read past their end."""
    for name in ("linear_nll", "linear_nll_back"):
        body = method(name)
        assert body.index("head_sizes(w, x, labels, b, trans)") < body.index("ccall")
    assert "length(lse) == 2N " in method("linear_nll_back") and "length(count) == 1" in method("linear_nll_back")
    sizes = method("head_sizes")
    for what in ("ndims(w) == 2", "size(x, 1) == H", "length(labels) == N", "length(b) == V"):
        assert what in sizes
