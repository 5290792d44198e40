"""GPU: the example runs the latent-attention operators beside the codec."""
import importlib.util
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_latent_context_example(dev):
    spec = importlib.util.spec_from_file_location("latent_context", os.path.join(ROOT, "examples", "latent_context.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["latent_context"] = mod
    spec.loader.exec_module(mod)
    event = mod.main(["--width", "64", "--height", "64", "--packets", "3", "--window-packets", "2", "--sinks", "16"])
    tokens = event["tokens_per_packet"]
    assert tokens == 64 and event["status"] == 0 and event["finite"]
    # the branch holds the I packet and three P packets, the released streams nothing
    assert event["lengths"] == [0, 4 * tokens, 0]
    assert 0 < event["pages_kept"] < event["pages_used"] and event["pages_lowest"]
    assert event["trials_differ"] > 0  # different QPs, different features
    assert len(event["bytes"]) == 6 and min(event["bytes"]) > 0
