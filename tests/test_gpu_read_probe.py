"""bench.py --read-probe, on a smaller buffer: every probe runs and prints its line."""
import json

import pytest

import bench

pytestmark = pytest.mark.gpu


def test_read_probe(monkeypatch, capsys):
    monkeypatch.setattr(bench, "READ_PROBE_BYTES", 64 << 20)
    bench.read_probe()
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    kinds = [line["probe"] for line in lines]
    assert [kinds.count(k) for k in ("read", "copy", "read_one_launch", "empty_kernel")] == [20, 1, 8, 3]
    assert all(v > 0 for line in lines for v in line.values() if not isinstance(v, str))
