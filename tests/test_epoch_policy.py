"""Host logic of the epoch runners that needs no GPU."""
import os
import subprocess
import sys

import pytest

from neutronbench_amd import epoch


def test_graph_mode_picked_by_batches_in_flight_and_feature_cache():
    """nts_batch_builder_use_graph value of the epoch loops: an explicit value is passed through; True
    picks the one recorded chain with several batches in flight, and with one batch in flight the
    second graph beside the gather."""
    assert epoch.graph_mode(True, 1, 0.2) == 3
    assert epoch.graph_mode(True, 1, 0.0) == 3
    assert epoch.graph_mode(True, 1) == 3
    for p in (2, 3, 4, 6):
        assert epoch.graph_mode(True, p, 0.2) == 1
        assert epoch.graph_mode(True, p, 0.0) == 1
    for explicit in (0, 1, 2, 3):
        assert epoch.graph_mode(explicit, 1, 0.2) == explicit
        assert epoch.graph_mode(explicit, 4, 0.0) == explicit
    assert epoch.graph_mode(False, 1, 0.2) == 0


def test_every_configuration_names_what_the_native_driver_needs():
    for name, cfg in epoch.CONFIGS.items():
        for key in ("V", "E", "F", "hidden", "classes", "fanout", "batch", "train", "seed", "cache"):
            assert key in cfg, (name, key)
        assert cfg["hidden"] % max(cfg.get("heads", 0), 1) == 0
        assert all(f != 0 for f in cfg["fanout"]) and 1 <= len(cfg["fanout"]) <= 8


@pytest.mark.parametrize("option", [["--native"], ["--write-inputs", "inputs"]])
def test_the_native_driver_takes_float_features_only(option, tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(epoch.__file__)))
    env = {**os.environ, "PYTHONPATH": root}
    got = subprocess.run([sys.executable, "-m", "neutronbench_amd.epoch", "--config", "arxiv", "--features", "mxfp4", *option],
                         cwd=tmp_path, env=env, capture_output=True, text=True)
    assert got.returncode == 2 and "--features f32" in got.stderr and not os.listdir(tmp_path)
