"""Options of python -m pdscope_amd.compare (CPU): what reaches the measured session."""
import json

import pytest

from pdscope_amd import compare


@pytest.mark.parametrize("given,want", [([], None), (["--int4-group", "32"], 32), (["--int4-group", "64"], 64),
                                        (["--int4-group", "128"], 128)])
def test_int4_group(given, want, monkeypatch, tmp_path, capsys):
    seen = {}

    def run(model, specs, **kw):
        seen.update(kw, model=model, specs=specs)
        return dict(status="completed")

    monkeypatch.setattr(compare, "random_qwen3_moe", lambda layers, seed: (layers, seed))
    monkeypatch.setattr(compare, "run", run)
    compare.main(["--random-layers", "2", "--seed", "5", "--output", str(tmp_path / "result.json"), *given])
    assert seen["model"] == (2, 5) and seen["config"]["int4_group"] == want
    assert seen.get("int4_group") == want and ("int4_group" in seen) == (want is not None)
    assert json.loads(capsys.readouterr().out)["status"] == "completed"


@pytest.mark.parametrize("given", [["--int4-group", "16"], ["--int4-group", "0"], ["--int4-group"]])
def test_groups_that_a_matrix_cannot_have(given, tmp_path, capsys):
    with pytest.raises(SystemExit):
        compare.main(["--random-layers", "2", "--output", str(tmp_path / "result.json"), *given])
    assert "--int4-group" in capsys.readouterr().err
