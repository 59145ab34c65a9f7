"""What the layer and model launchers refuse before they touch a GPU."""
import os
import subprocess
import sys

import pytest

ENGINE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pim-dl-asplos_b200", "inference_engine")


@pytest.mark.parametrize("driver", ["run_layer.py", "run_model.py"])
@pytest.mark.parametrize("flags", [["--window", "32"], ["--sinks", "1"], ["--window", "0", "--sinks", "2"]])
def test_a_window_needs_the_dense_kernels(driver, flags):
    r = subprocess.run([sys.executable, os.path.join(ENGINE, driver), "--transformer_config_file", "none.yaml", *flags], capture_output=True, text=True, timeout=300)
    assert r.returncode == 2 and "--dense_kernels" in r.stderr


@pytest.mark.parametrize("flags", [[], ["--window", "-1"], ["--dense_kernels", "--window", "32", "--sinks", "1"], ["--dense_kernels"]])
def test_the_others_are_taken(monkeypatch, flags):
    monkeypatch.syspath_prepend(ENGINE)
    import run_layer
    monkeypatch.setattr(sys, "argv", ["run_layer.py", "--transformer_config_file", "none.yaml", *flags])
    args = run_layer.parse_args()
    assert args.dense_kernels == ("--dense_kernels" in flags)
