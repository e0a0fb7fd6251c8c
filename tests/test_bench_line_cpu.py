"""The benchmark's result line: short enough that the end of a log holds it whole, with nothing of the contract left out."""
import json
import os

import bench


def test_result_line_is_short_and_details_are_whole(tmp_path):
    line = {key: "x" * 60 for key in bench.LINE_KEYS}
    line.update(configs={f"row{i}": {"ms": 1.0, "note": "y" * 700} for i in range(25)}, side={"a": "z" * 700}, configs_summary={"rows": 25})
    out, details = tmp_path / "line", tmp_path / "details.json"
    fd = os.open(out, os.O_WRONLY | os.O_CREAT)
    bench.emit(fd, line, str(details))
    os.close(fd)
    text = out.read_text()
    assert text.endswith("\n") and text.count("\n") == 1 and len(text) <= bench.LINE_LIMIT + 100
    short = json.loads(text)
    assert all(short[key] == line[key] for key in bench.LINE_KEYS) and short["configs_summary"] == {"rows": 25}
    assert short["in_details"] == ["configs"] and "configs" not in short and short["side"] == line["side"]
    assert json.loads(details.read_text()) == line


def test_result_line_that_fits_is_left_alone(tmp_path):
    out = tmp_path / "line"
    fd = os.open(out, os.O_WRONLY | os.O_CREAT)
    bench.emit(fd, {"metric": "m", "value": 1.0, "parity": {"worst": 0.0}})
    os.close(fd)
    assert json.loads(out.read_text()) == {"metric": "m", "value": 1.0, "parity": {"worst": 0.0}}
