"""The benchmark's reference arm measures the reference or nothing."""
import argparse
import json

import bench
from oracle.oracle import Oracle


def test_reference_arm_without_the_reference(monkeypatch, capsys):
    monkeypatch.setattr(Oracle, "reference_available", staticmethod(lambda: False))
    monkeypatch.delenv("RANK", raising=False)
    bench.run_reference(argparse.Namespace(gpus=1, steps=2, warmup=1))
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
