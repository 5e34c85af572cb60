"""Arguments of the operator benchmark that no operator has are refused before anything is measured."""
import pytest

from uniserve_v1_b200.tools import opbench


@pytest.mark.parametrize("op", ["decode", "scored", "rank-decode"])
@pytest.mark.parametrize("kv", ["int8", "int4"])
def test_integer_pages_are_of_scored_decode_alone(op, kv, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["opbench", op, "--kv", kv])
    monkeypatch.setattr(opbench, "peaks", lambda: pytest.fail("went on to measure"))
    with pytest.raises(SystemExit) as end:
        opbench.main()
    assert end.value.code == 2 and f"{kv} pages" in capsys.readouterr().err
