"""run_all.py --item_bits: refused before any training where it cannot be, named in every record."""
import importlib.util
import json

import pytest

from conftest import PKG


@pytest.fixture
def run_all(monkeypatch):
    spec = importlib.util.spec_from_file_location("run_all", PKG / "run_all.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_4_bit_items_on_the_cpu_are_refused_before_training(run_all, monkeypatch, tmp_path, capsys):
    def trained(*args):
        raise AssertionError("a model was trained")

    monkeypatch.setattr(run_all, "train_bpr", trained)
    with pytest.raises(SystemExit) as stop:
        run_all.main(["--quick", "--device", "cpu", "--item_bits", "4", "--skip-check",
                      "--output", str(tmp_path / "r.json")])
    assert stop.value.code == 2 and "ROCm device" in capsys.readouterr().err
    assert not (tmp_path / "r.json").exists()


def test_records_name_the_items_width(run_all, tmp_path):
    out = tmp_path / "r.json"
    assert run_all.main(["--quick", "--epochs", "0", "--device", "cpu", "--skip-check", "--models",
                         "lightgcn", "--output", str(out)]) == 0
    assert [r["item_bits"] for r in json.loads(out.read_text())] == [32]


@pytest.mark.gpu
def test_records_on_the_device(cuda, run_all, tmp_path):
    out = tmp_path / "r.json"
    assert run_all.main(["--quick", "--epochs", "0", "--device", "cuda", "--skip-check", "--models",
                         "lightgcn", "--item_bits", "4", "--output", str(out)]) == 0
    rec, = json.loads(out.read_text())
    assert rec["item_bits"] == 4 and rec["test_metrics"]
