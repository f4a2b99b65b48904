"""examples/graph_layer.py: the dense operators and the SpMM together.  The loss starts at ln(16) (the classifier
starts near zero) and falls; 8-bit serving follows the 16-bit layer: codes are within 1/254 of a row's and a channel's
largest value, so logits of 64 terms are off by a few percent at most."""
import math
import os
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_layer_trains_and_serves():
    print("example", flush=True)
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import graph_layer
    finally:
        sys.path.pop(0)
    got = graph_layer.run(nodes=4096, width=64, types=512, steps=40)
    print(got, flush=True)
    assert abs(got["first"] - math.log(16)) < 0.5
    assert got["last"] < 0.5 * got["first"]
    assert got["off"] < 0.05 and got["same"] > 0.95 and got["right"] > 0.8
